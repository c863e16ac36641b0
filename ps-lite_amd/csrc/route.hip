// Tokens to the experts they chose, and back (gfx950). T tokens name K experts each; choice i = t*K + j. The choices are
// sorted by expert, stably, so that every expert finds its rows back to back; a token's row is copied to its K places, and the
// experts' answers come back as a weighted sum:
//     place[i]      = #{choices of lower experts} + #{earlier choices of the same expert}
//     rows[place]   = x[t]                              its gradient: dx[t] = sum_j drows[place[t,j]]
//     y[t]          = sum_j w[t,j] answers[place[t,j]]  its gradient: danswers[place] = w dy[t], dw[t,j] = <dy[t], answers[place]>
// Everything but the sort goes token by token: a token's own row is read or written once, its K others once each, nothing is
// summed by more than one wavefront, and no sum depends on the order in which workgroups run. (The gradient of y reads a token's row once
// for every wavefront that its choices are shared out to, and once for every choice where it is longer than 256 vectors of 16 bytes.)
#include <hip/hip_runtime.h>

#include "host_common.h"
#include "lanes.h"
#include "row_types.h"

namespace pskv {
namespace {

// --- sorting by expert -------------------------------------------------------------------------------------------

constexpr unsigned kSortBlock = 1024;
constexpr unsigned kSortWaves = kSortBlock / 64;
// Up to so many counts, every workgroup adds up the tiles' for itself; beyond, a launch of its own does. Both sides, with the
// launch's own start of about 1 us: 64 tiles of 257 counts 14.5 and 16.9 us, 128 of 257 19.4 and 18.6, 32 of 1,025 19.0 and 18.3,
// 512 of 257 61 and 36, 64 of 2,048 32 and 22.
constexpr uint64_t kSortFew = 32768;
constexpr unsigned kSortBins = PSKV_ROUTE_MAX_EXPERTS + 1;  // the last one in use: choices that are not here

template <typename I>
__device__ __forceinline__ unsigned bin_of(const I* experts, uint64_t i, unsigned E) {
  const I e = experts[i];
  return e >= 0 && e < (I)E ? (unsigned)e : E;
}

// How many choices of every bin a tile has: counts[tile][bin].
template <typename I, unsigned ITEMS>
__global__ __launch_bounds__(kSortBlock) void k_route_count(const I* __restrict__ experts, uint64_t n, unsigned E,
                                                             unsigned* __restrict__ counts) {
  __shared__ unsigned hist[kSortBins];
  for (unsigned e = threadIdx.x; e <= E; e += kSortBlock) hist[e] = 0;
  const uint64_t first = (uint64_t)blockIdx.x * (kSortBlock * ITEMS) + threadIdx.x;
  unsigned bin[ITEMS];
#pragma unroll
  for (unsigned s = 0; s < ITEMS; ++s)
    bin[s] = first + s * kSortBlock < n ? bin_of(experts, first + s * kSortBlock, E) : kSortBins;
  __syncthreads();
#pragma unroll
  for (unsigned s = 0; s < ITEMS; ++s)
    if (bin[s] < kSortBins) atomicAdd(&hist[bin[s]], 1u);
  __syncthreads();
  for (unsigned e = threadIdx.x; e <= E; e += kSortBlock) counts[(uint64_t)blockIdx.x * (E + 1) + e] = hist[e];
}

// What every tile's choices of a bin follow, in place, and behind the last tile the bins' totals. A workgroup takes 64 bins, a lane
// to each; its wavefronts share the tiles out, add up their parts, and go through them once more from where the parts before end.
__global__ __launch_bounds__(kSortBlock) void k_route_scan(unsigned* __restrict__ counts, unsigned tiles, unsigned bins) {
  __shared__ unsigned part[kSortWaves][64];
  const unsigned wave = threadIdx.x >> 6, lane = threadIdx.x & 63, e = blockIdx.x * 64 + lane;
  const unsigned each = (tiles + kSortWaves - 1) / kSortWaves;
  const unsigned first = wave * each < tiles ? wave * each : tiles, end = tiles - first < each ? tiles : first + each;
  constexpr unsigned kAhead = 16;
  auto pass = [&](unsigned run, auto write) {
    for (unsigned t0 = first; t0 < end; t0 += kAhead) {
      unsigned c[kAhead];
#pragma unroll
      for (unsigned a = 0; a < kAhead; ++a) c[a] = t0 + a < end && e < bins ? counts[(uint64_t)(t0 + a) * bins + e] : 0;
#pragma unroll
      for (unsigned a = 0; a < kAhead; ++a) {
        if (decltype(write)::value && t0 + a < end && e < bins) counts[(uint64_t)(t0 + a) * bins + e] = run;
        run += c[a];
      }
    }
    return run;
  };
  part[wave][lane] = pass(0, std::false_type());
  __syncthreads();
  unsigned run = 0, all = 0;
#pragma unroll
  for (unsigned w = 0; w < kSortWaves; ++w) {
    run += w < wave ? part[w][lane] : 0;
    all += part[w][lane];
  }
  pass(run, std::true_type());
  if (wave == 0 && e < bins) counts[(uint64_t)tiles * bins + e] = all;
}

// Places of a tile's choices. A wavefront owns neighbouring ones and takes them 64 at a time: lanes of the same bin find each
// other by comparing the bits of their bins, so a choice's rank among its wavefront's is known without atomics; ranks begin
// where the earlier wavefronts', tiles' and bins' choices end. 16 choices take 2.9 us; with their counts, in a graph of sorts, 15,009 of
// 64 experts 7.0 and 262,144 of 256 13.3 (in a trace the kernels' own times add up to 7.7 to 8.3 and 16.0): a chain of steps that each wait for the one before, on as many compute units as there are tiles (every workgroup
// counting all choices itself instead of a launch for the counts: twice the time where half of them are of one expert, for the atomics
// on one counter).
template <typename I, unsigned ITEMS>
__global__ __launch_bounds__(kSortBlock) void k_route_place(const I* __restrict__ experts, uint64_t n, unsigned E,
                                                             const unsigned* __restrict__ counts, unsigned tiles,
                                                             bool scanned, int* __restrict__ order,
                                                             int* __restrict__ place, int* __restrict__ offsets) {
  __shared__ unsigned short mine[kSortWaves][kSortBins];  // of a wavefront, then of those before it
  __shared__ unsigned total[kSortBins], base[kSortBins];  // of a bin in all tiles, in the tiles before
  __shared__ unsigned sums[kSortWaves];
  const unsigned bins = E + 1, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const uint64_t first = (uint64_t)blockIdx.x * (kSortBlock * ITEMS) + wave * (64 * ITEMS) + lane;
  unsigned bin[ITEMS], rank[ITEMS];
#pragma unroll
  for (unsigned s = 0; s < ITEMS; ++s) bin[s] = first + s * 64 < n ? bin_of(experts, first + s * 64, E) : bins;
  for (unsigned e = lane; e < bins; e += 64) mine[wave][e] = 0;
  for (unsigned e = threadIdx.x; e < bins; e += kSortBlock) {
    total[e] = tiles > 1 && scanned ? counts[(uint64_t)tiles * bins + e] : 0;
    base[e] = tiles > 1 && scanned ? counts[(uint64_t)blockIdx.x * bins + e] : 0;
  }
  __syncthreads();
  if (tiles > 1 && !scanned) {
    // the counts lie tile by tile: a thread's steps through them are 1,024 apart
    const unsigned all = tiles * bins, before = blockIdx.x * bins, hop = kSortBlock % bins;
    unsigned e = threadIdx.x % bins;
    constexpr unsigned kAhead = 8;
    for (unsigned i0 = threadIdx.x; i0 < all; i0 += kAhead * kSortBlock) {
      unsigned c[kAhead];
#pragma unroll
      for (unsigned a = 0; a < kAhead; ++a) c[a] = i0 + a * kSortBlock < all ? counts[i0 + a * kSortBlock] : 0;
#pragma unroll
      for (unsigned a = 0; a < kAhead; ++a) {
        if (c[a]) {
          atomicAdd(&total[e], c[a]);
          if (i0 + a * kSortBlock < before) atomicAdd(&base[e], c[a]);
        }
        e += hop;
        if (e >= bins) e -= bins;
      }
    }
  }
  const unsigned bits = 32 - __builtin_clz(bins);
  const uint64_t before = (1ull << lane) - 1;
  uint64_t same[ITEMS];  // the lanes of the same bin
#pragma unroll
  for (unsigned s = 0; s < ITEMS; ++s) same[s] = ~0ull;
  for (unsigned b = 0; b < bits; ++b) {
#pragma unroll
    for (unsigned s = 0; s < ITEMS; ++s) {
      const int bit = (int)(bin[s] << (31 - b)) >> 31;  // 0 or all ones
      const uint64_t ones = __ballot(bit != 0);
      same[s] &= ~(ones ^ (uint64_t)(int64_t)bit);
    }
  }
#pragma unroll
  for (unsigned s = 0; s < ITEMS; ++s) {
    if (bin[s] < bins) {
      const unsigned so_far = mine[wave][bin[s]];
      rank[s] = so_far + __popcll(same[s] & before);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if ((same[s] >> lane) == 1) mine[wave][bin[s]] = (unsigned short)(so_far + __popcll(same[s]));
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  __syncthreads();
  // where every bin begins: the totals summed up over the bins, some to a thread
  constexpr unsigned kPer = (kSortBins + kSortBlock - 1) / kSortBlock;
  const unsigned per = (bins + kSortBlock - 1) / kSortBlock;
  unsigned amount[kPer], all = 0;
#pragma unroll
  for (unsigned q = 0; q < kPer; ++q) {
    const unsigned e = threadIdx.x * per + q;
    amount[q] = 0;
    if (q < per && e < bins) {
      unsigned run = 0;
#pragma unroll
      for (unsigned w = 0; w < kSortWaves; ++w) {
        const unsigned c = mine[w][e];
        mine[w][e] = (unsigned short)run;
        run += c;
      }
      amount[q] = tiles > 1 ? total[e] : run;
    }
    all += amount[q];
  }
  unsigned inc = all;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned up = __shfl_up(inc, o);
    inc += lane >= (unsigned)o ? up : 0;
  }
  if (lane == 63) sums[wave] = inc;
  __syncthreads();
  unsigned run = inc - all;
  for (unsigned w = 0; w < wave; ++w) run += sums[w];
#pragma unroll
  for (unsigned q = 0; q < kPer; ++q) {
    const unsigned e = threadIdx.x * per + q;
    if (q < per && e < bins) {
      base[e] += run;
      if (blockIdx.x == 0) offsets[e] = (int)run;
    }
    run += amount[q];
  }
  __syncthreads();
#pragma unroll
  for (unsigned s = 0; s < ITEMS; ++s) {
    if (bin[s] >= bins) continue;
    const uint64_t i = first + s * 64;
    const unsigned p = base[bin[s]] + mine[wave][bin[s]] + rank[s];
    const bool here = bin[s] < E;
    place[i] = here ? (int)p : -1;
    if (p < n) order[p] = here ? (int)i : -1;  // (always, but where experts or counts change under the call)
  }
}

// --- rows out and back -------------------------------------------------------------------------------------------

// Where there are many tokens and rows are whole lines, all three kernels move what they have to and nothing else (read and written at the
// memory: 1.00 of it, the gradient up to 256 vectors a row), so the memory bounds them. Rows that begin and end inside lines move some
// 10 % more (3 x 5,003 rows of 1,001 float16: 10.8 MB read for 10.0 out, 26.4 for 24.0 back; the gradient of 6 x 1,999 of 777 float32, whose token's
// row is read by every wavefront that has some of its choices: 45.5 for 39.9), and their last elements, fewer than a vector, are asked for
// choice by choice, each behind the one before. 32,768 x 8 rows of 2,048 bf16 out at 5.3 TB/s (1.2 GB in 229 us; rows of 4 KB that go to eight places) and
// back at 5.8 (210 us), the gradient of 16,384 x 4 at 5.5 (111 us). Calls that move more than the memory-side cache holds go
// past it (back: 280 -> 211 us; the gradient and the sum of its rows 178 -> 165); smaller ones leave it their rows, which the
// next call wants (36 MB past it: 8.4 -> 10.8 us out, 8.9 -> 9.7 back).
constexpr unsigned kRowBlock = 256;

// (Kernels with up to 104 bytes of arguments that do not ask for the size of their grid take the calling thread 2.7 us to launch, others 3.3.)
struct RowArgs {
  uint64_t token_stride, row_stride;  // elements
  uint32_t tokens, k, rows;           // rows: of the sorted side
  uint32_t choices, lanes_log2;
  uint32_t groups;  // workgroups of the launch
};

// The token of a lane; where a wavefront or more serves one, the compiler is told that all lanes have the same, so that places and
// weights are loaded once per wavefront.
template <bool ONE>
__device__ __forceinline__ uint64_t token_of(uint64_t t) {
  if (!ONE) return t;
  return (uint64_t)__builtin_amdgcn_readfirstlane((int)(t >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)t);
}

template <typename T, bool ONE, bool PAST>
__global__ __launch_bounds__(kRowBlock) void k_route_rows(const T* __restrict__ x, const int* __restrict__ place,
                                                           T* __restrict__ out, RowArgs a) {
  using Vec = typename Row<T>::Vec;
  constexpr unsigned W = Row<T>::kWide;
  const unsigned lanes = 1u << a.lanes_log2;
  const uint64_t per = (uint64_t)a.groups * (kRowBlock >> a.lanes_log2);
  for (uint64_t t = token_of<ONE>(((uint64_t)blockIdx.x * kRowBlock + threadIdx.x) >> a.lanes_log2); t < a.tokens; t += per) {
    const T* from = x + t * a.token_stride;
    const int* at = place + t * a.choices;
    for (uint64_t c = (uint64_t)(threadIdx.x & (lanes - 1)) * W; c < a.k; c += (uint64_t)lanes * W) {
      if (c + W <= a.k) {
        const Vec v = get<false>(from + c);
        for (unsigned j = 0; j < a.choices; ++j) {
          const uint64_t p = (uint64_t)(int64_t)at[j];
          if (p < a.rows) put<PAST>(out + p * a.row_stride + c, v);
        }
      } else {
        for (unsigned j = 0; j < a.choices; ++j) {
          const uint64_t p = (uint64_t)(int64_t)at[j];
          if (p < a.rows)
            for (uint64_t i = c; i < a.k; ++i) out[p * a.row_stride + i] = from[i];
        }
      }
    }
  }
}

// Eight answers are asked for at a time. A choice that is not here reads row 0, whose elements are replaced by zeros.
template <typename T, bool ONE, bool PAST>
__global__ __launch_bounds__(kRowBlock) void k_route_sum(const T* __restrict__ rows, const int* __restrict__ place,
                                                          const float* __restrict__ weights, T* __restrict__ out, RowArgs a) {
  using Vec = typename Row<T>::Vec;
  constexpr unsigned W = Row<T>::kWide, kAhead = 8;
  const unsigned lanes = 1u << a.lanes_log2;
  const uint64_t per = (uint64_t)a.groups * (kRowBlock >> a.lanes_log2);
  for (uint64_t t = token_of<ONE>(((uint64_t)blockIdx.x * kRowBlock + threadIdx.x) >> a.lanes_log2); t < a.tokens; t += per) {
    const int* at = place + t * a.choices;
    const float* w = weights ? weights + t * a.choices : nullptr;
    T* to = out + t * a.token_stride;
    for (uint64_t c = (uint64_t)(threadIdx.x & (lanes - 1)) * W; c < a.k; c += (uint64_t)lanes * W) {
      float sum[W] = {};
      if (c + W <= a.k) {
        auto some = [&](unsigned j0, auto count) {
          constexpr unsigned N = decltype(count)::value;
          Vec v[N];
          bool here[N];
#pragma unroll
          for (unsigned j = 0; j < N; ++j) {
            const uint64_t p = (uint64_t)(int64_t)at[j0 + j];
            here[j] = p < a.rows;
            v[j] = get<PAST>(rows + (here[j] ? p : 0) * a.row_stride + c);
          }
#pragma unroll
          for (unsigned j = 0; j < N; ++j) {
            const float f = !here[j] ? 0.0f : w ? w[j0 + j] : 1.0f;
#pragma unroll
            for (unsigned i = 0; i < W; ++i) sum[i] = __builtin_fmaf(f, here[j] ? (float)v[j][i] : 0.0f, sum[i]);
          }
        };
        unsigned j = 0;
        for (; j + kAhead <= a.choices; j += kAhead) some(j, std::integral_constant<unsigned, kAhead>());
        if (a.choices & 4) some(j, std::integral_constant<unsigned, 4>()), j += 4;
        if (a.choices & 2) some(j, std::integral_constant<unsigned, 2>()), j += 2;
        if (a.choices & 1) some(j, std::integral_constant<unsigned, 1>());
        Vec v;
#pragma unroll
        for (unsigned i = 0; i < W; ++i) v[i] = (T)sum[i];
        put<PAST>(to + c, v);
      } else {
        const unsigned wide = (unsigned)(a.k - c);
        for (unsigned j = 0; j < a.choices; ++j) {
          const uint64_t p = (uint64_t)(int64_t)at[j];
          if (p >= a.rows) continue;
          const float f = w ? w[j] : 1.0f;
#pragma unroll
          for (unsigned i = 0; i < W; ++i)
            if (i < wide) sum[i] = __builtin_fmaf(f, (float)rows[p * a.row_stride + c + i], sum[i]);
        }
#pragma unroll
        for (unsigned i = 0; i < W; ++i)
          if (i < wide) to[c + i] = (T)sum[i];
      }
    }
  }
}

// At most a wavefront per token, so that the products' sums need no other than its own lanes. A lane keeps its part of the
// token's gradient, NV vectors of it, for all its choices (`share` of them, all where there are many tokens), and asks for four
// vectors of the answers at once, of 4 / NV choices. Rows of more than 4 x 64 vectors (LONG) go piece by piece, and the token's
// gradient is asked for anew with every choice: 8,192 x 4 of 4,096 bf16 128 us, of 2,048 float32 123, 487 MB read for 336 (some of it again from
// the caches), where 16,384 x 4 of 2,048 bf16, as many bytes, take 111.
constexpr unsigned kKept = 4;

template <typename T, bool ONE, bool PAST, unsigned NV, bool LONG>
__global__ __launch_bounds__(kRowBlock) void k_route_sum_grad(const T* __restrict__ grad, const T* __restrict__ rows,
                                                               const int* __restrict__ place,
                                                               const float* __restrict__ weights, T* __restrict__ grad_rows,
                                                               uint64_t grad_row_stride, float* __restrict__ grad_weights,
                                                               unsigned share, RowArgs a) {
  using Vec = typename Row<T>::Vec;
  constexpr unsigned W = Row<T>::kWide, C = kKept / NV;
  const unsigned lanes = 1u << a.lanes_log2, lane = threadIdx.x & (lanes - 1);
  const uint64_t per = kRowBlock >> a.lanes_log2;
  const uint64_t wide = (uint64_t)lanes * W, whole = (uint64_t)a.k / W * W;  // elements of a vector for all lanes; of whole vectors
  const unsigned parts = (a.choices + share - 1) / share;
  const uint64_t units = (uint64_t)a.tokens * parts;
  // (lanes of one unit add up together, and leave together)
  for (uint64_t u = token_of<ONE>(blockIdx.x * per + (threadIdx.x >> a.lanes_log2)); u < units; u += a.groups * per) {
    const unsigned t = (unsigned)u / parts, j0 = ((unsigned)u - t * parts) * share;
    const unsigned end = a.choices - j0 < share ? a.choices : j0 + share;
    const T* g = grad + t * a.token_stride;
    const int* at = place + (uint64_t)t * a.choices;
    const float* w = weights + (uint64_t)t * a.choices;
    typedef uint32_t Words __attribute__((ext_vector_type(4)));
    Words kept[NV] = {};
    auto fetch = [&](uint64_t c0) {
#pragma unroll
      for (unsigned q = 0; q < NV; ++q)
        if (c0 + q * wide < whole) kept[q] = __builtin_bit_cast(Words, get<false>(g + c0 + q * wide));
    };
    if (!LONG) fetch(lane * W);
    for (unsigned j = j0; j < end; j += C) {
      // (the gradient is kept as it is in memory: as numbers, for all choices, it would take twice the registers, and fewer wavefronts
      // would be at work: 109 us became 124 for 16,384 x 4 answers of 2,048 bf16)
      Vec d[NV];
#pragma unroll
      for (unsigned q = 0; q < NV; ++q) {
        asm volatile("" : "+v"(kept[q]));
        d[q] = __builtin_bit_cast(Vec, kept[q]);
      }
      Vec v[C][NV];
      uint64_t p[C];
      float f[C], sum[C];
#pragma unroll
      for (unsigned i = 0; i < C; ++i) {
        const bool is = j + i < end;
        p[i] = is ? (uint64_t)(int64_t)at[j + i] : ~0ull;
        f[i] = is ? w[j + i] : 0.0f;
        sum[i] = 0.0f;
      }
      for (uint64_t c0 = lane * W; c0 < whole; c0 += NV * wide) {
#pragma unroll
        for (unsigned i = 0; i < C; ++i)
#pragma unroll
          for (unsigned q = 0; q < NV; ++q)
            if (p[i] < a.rows && c0 + q * wide < whole) v[i][q] = get<PAST>(rows + p[i] * a.row_stride + c0 + q * wide);
        if (LONG) {
          fetch(c0);
#pragma unroll
          for (unsigned q = 0; q < NV; ++q) d[q] = __builtin_bit_cast(Vec, kept[q]);
        }
#pragma unroll
        for (unsigned i = 0; i < C; ++i)
#pragma unroll
          for (unsigned q = 0; q < NV; ++q)
            if (p[i] < a.rows && c0 + q * wide < whole) {
              Vec o;
#pragma unroll
              for (unsigned e = 0; e < W; ++e) {
                sum[i] = __builtin_fmaf((float)d[q][e], (float)v[i][q][e], sum[i]);
                o[e] = (T)(f[i] * (float)d[q][e]);
              }
              put<PAST>(grad_rows + p[i] * grad_row_stride + c0 + q * wide, o);
            }
        if (!LONG) break;
      }
#pragma unroll
      for (unsigned i = 0; i < C; ++i) {
        if (p[i] < a.rows)
          for (uint64_t c = whole + lane; c < a.k; c += lanes) {
            sum[i] = __builtin_fmaf((float)g[c], (float)rows[p[i] * a.row_stride + c], sum[i]);
            grad_rows[p[i] * grad_row_stride + c] = (T)(f[i] * (float)g[c]);
          }
        if (ONE) {
          sum[i] = sum_along(sum[i], 0);
        } else {
          for (unsigned o = lanes >> 1; o > 0; o >>= 1) sum[i] += __shfl_xor(sum[i], o);
        }
        if (lane == lanes - 1 && j + i < end) grad_weights[(uint64_t)t * a.choices + j + i] = sum[i];
      }
    }
  }
}

// --- the host's checks -------------------------------------------------------------------------------------------

// What every call between tokens and sorted rows refuses. PSKV_OK: it may run.
int check_rows(int type, uint64_t tokens, uint64_t choices, uint64_t rows, uint64_t k) {
  if (!type_bytes(type)) return set_error(PSKV_EINVAL, "type %d: PSKV_F32, PSKV_F16 or PSKV_BF16", type);
  if (choices == 0) return set_error(PSKV_EINVAL, "a token chooses at least one expert");
  if (k == 0 || k > (1ull << 30)) return set_error(PSKV_EINVAL, "rows of 1 to 2^30 elements");
  if (tokens > 0x7fffffffull || choices > 0x7fffffffull || tokens * choices > 0x7fffffffull || rows > 0x7fffffffull)
    return set_error(PSKV_EINVAL, "2^31 - 1 choices and rows at most");
  return PSKV_OK;
}

int check_stride(const char* what, uint64_t n, uint64_t k, uint64_t stride, bool written) {
  if (stride > (1ull << 40)) return set_error(PSKV_EINVAL, "%s: rows 2^40 elements apart at most", what);
  if (written && n > 1 && stride < k) return set_error(PSKV_EINVAL, "%s: rows that are written lie upon each other", what);
  return PSKV_OK;
}

// How a sort is cut into tiles: 1, 2 or 4 choices to each of a workgroup's 1,024 lanes. One tile, and one launch, up to 4,096. From
// there on as small tiles as there may be, for a tile's steps are what takes the time (in a graph of sorts, 15,009 choices of 64 experts: 6.8 us
// with one choice to a lane, 7.5 with two, 9.5 with four; 262,144 of 256: 13.3 with two, 13.7 with four), until adding up the tiles' counts
// takes longer (524,288 of 256: 21.2, 15.4, 16.9; 1,048,576 of 64: two 22.9, four 16.3).
struct SortCut {
  unsigned items;
  uint64_t tiles;
  explicit SortCut(uint64_t n) {
    items = n <= 4096 ? (n <= 1024 ? 1 : n <= 2048 ? 2 : 4) : n <= 131072 ? 1 : n <= 524288 ? 2 : 4;
    tiles = n ? (n + kSortBlock * items - 1) / (kSortBlock * items) : 1;
  }
};

// Most lanes of a token whose row is copied or summed: a workgroup's where there are few tokens (512 x 4 rows of 4,096 bf16: 5.9 us,
// with two wavefronts 6.7), two wavefronts otherwise (32,768 x 8 of 2,048: 236 and 227).
unsigned lanes_of(uint64_t tokens) { return tokens < 2048 ? kRowBlock : 128; }

RowArgs row_args(uint64_t tokens, uint64_t choices, uint64_t rows, uint64_t k, uint64_t token_stride, uint64_t row_stride,
                 int type, unsigned most_lanes) {
  const uint64_t wide = 16 / type_bytes(type);
  const unsigned lanes = lanes_for((k + wide - 1) / wide, most_lanes);
  const unsigned lanes_log2 = (unsigned)__builtin_ctz(lanes);
  return RowArgs{token_stride, row_stride, (uint32_t)tokens, (uint32_t)k, (uint32_t)rows, (uint32_t)choices, lanes_log2,
                 grid_for(tokens, kRowBlock >> lanes_log2, 1u << 22)};
}

}  // namespace
}  // namespace pskv

using namespace pskv;

#define RETURN_IF(call)     \
  do {                      \
    const int rc_ = (call); \
    if (rc_) return rc_;    \
  } while (0)

extern "C" size_t pskv_route_room(size_t n, size_t E) {
  if (n > 0x7fffffffull || E > PSKV_ROUTE_MAX_EXPERTS) return 0;
  const SortCut cut(n);
  return cut.tiles == 1 ? 0 : (cut.tiles + 1) * (E + 1) * sizeof(unsigned);
}

extern "C" int pskv_route_sort(int device, void* stream, const void* experts, int index_bits, size_t n, size_t E,
                               int32_t* order, int32_t* place, int32_t* offsets, void* work, size_t work_bytes) {
  clear_error();
  if (index_bits != 32 && index_bits != 64) return set_error(PSKV_EINVAL, "experts are numbers of 32 or 64 bits");
  if (E == 0 || E > PSKV_ROUTE_MAX_EXPERTS)
    return set_error(PSKV_EINVAL, "%zu experts: 1 to %d", E, PSKV_ROUTE_MAX_EXPERTS);
  if (n > 0x7fffffffull) return set_error(PSKV_EINVAL, "2^31 - 1 choices at most");
  if (!offsets || (n && (!experts || !order || !place))) return set_error(PSKV_EINVAL, "null buffer");
  const size_t room = pskv_route_room(n, E);
  if (room && (!work || work_bytes < room || (reinterpret_cast<uintptr_t>(work) & 3)))
    return set_error(PSKV_EINVAL, "a sort of %zu choices takes %zu bytes of working memory, %zu given", n, room,
                     work ? work_bytes : (size_t)0);
  const struct {
    const void* at;
    uint64_t bytes;
  } used[5] = {{experts, n * (uint64_t)index_bits / 8}, {order, n * 4}, {place, n * 4}, {offsets, (E + 1) * 4}, {work, room}};
  for (int i = 0; i < 5; ++i)
    for (int j = i + 1; j < 5; ++j)
      if (overlap(used[i].at, used[i].bytes, used[j].at, used[j].bytes))
        return set_error(PSKV_EINVAL, "the experts, the answers and the working memory overlap");
  DeviceGuard guard(device);
  if (!guard.ok()) return set_error(PSKV_EHIP, "cannot select device %d", device);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const SortCut cut(n);
  const unsigned tiles = (unsigned)cut.tiles;
  const bool scanned = tiles * (E + 1) > kSortFew;
  unsigned* counts = static_cast<unsigned*>(work);
  auto go = [&](auto* e, auto items) {
    using I = std::remove_const_t<std::remove_pointer_t<decltype(e)>>;
    constexpr unsigned ITEMS = decltype(items)::value;
    if (tiles > 1) {
      hipLaunchKernelGGL((k_route_count<I, ITEMS>), dim3(tiles), dim3(kSortBlock), 0, st, e, (uint64_t)n, (unsigned)E, counts);
      if (scanned) hipLaunchKernelGGL(k_route_scan, dim3((unsigned)E / 64 + 1), dim3(kSortBlock), 0, st, counts, tiles, (unsigned)E + 1);
    }
    hipLaunchKernelGGL((k_route_place<I, ITEMS>), dim3(tiles), dim3(kSortBlock), 0, st, e, (uint64_t)n, (unsigned)E, counts, tiles,
                       scanned, order, place, offsets);
  };
  auto with_items = [&](auto* e) {
    if (cut.items == 1)
      go(e, std::integral_constant<unsigned, 1>());
    else if (cut.items == 2)
      go(e, std::integral_constant<unsigned, 2>());
    else
      go(e, std::integral_constant<unsigned, 4>());
  };
  if (index_bits == 64)
    with_items(static_cast<const int64_t*>(experts));
  else
    with_items(static_cast<const int32_t*>(experts));
  PSKV_HIP(hipGetLastError());
  return PSKV_OK;
}

extern "C" int pskv_route_rows(int device, void* stream, int type, const void* x, size_t x_stride, size_t tokens, size_t k,
                               const int32_t* place, size_t choices, void* rows, size_t rows_stride, size_t n_rows) {
  clear_error();
  RETURN_IF(check_rows(type, tokens, choices, n_rows, k));
  RETURN_IF(check_stride("x", tokens, k, x_stride, false));
  RETURN_IF(check_stride("rows", n_rows, k, rows_stride, true));
  if (tokens == 0 || n_rows == 0) return PSKV_OK;
  if (!x || !place || !rows) return set_error(PSKV_EINVAL, "null buffer");
  const size_t size = type_bytes(type);
  const RowSpan to{rows, n_rows, k, rows_stride, size};
  if (rows_overlap({x, tokens, k, x_stride, size}, to) || rows_overlap(stretch(place, tokens * choices * sizeof(int32_t)), to))
    return set_error(PSKV_EINVAL, "the rows that are written overlap what is read");
  DeviceGuard guard(device);
  if (!guard.ok()) return set_error(PSKV_EHIP, "cannot select device %d", device);
  const RowArgs a = row_args(tokens, choices, n_rows, k, x_stride, rows_stride, type, lanes_of(tokens));
  with_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    with_flag((1 + choices) * tokens * k * size > kPastBytes, [&](auto far) {
      constexpr bool PAST = decltype(far)::value;
      auto kernel = a.lanes_log2 >= 6 ? k_route_rows<T, true, PAST> : k_route_rows<T, false, PAST>;
      hipLaunchKernelGGL(kernel, dim3(a.groups), dim3(kRowBlock), 0,
                         static_cast<hipStream_t>(stream), static_cast<const T*>(x), place, static_cast<T*>(rows), a);
    });
  });
  PSKV_HIP(hipGetLastError());
  return PSKV_OK;
}

extern "C" int pskv_route_sum(int device, void* stream, int type, const void* rows, size_t rows_stride, size_t n_rows,
                              const int32_t* place, const float* weights, size_t choices, void* out, size_t out_stride,
                              size_t tokens, size_t k) {
  clear_error();
  RETURN_IF(check_rows(type, tokens, choices, n_rows, k));
  RETURN_IF(check_stride("rows", n_rows, k, rows_stride, false));
  RETURN_IF(check_stride("out", tokens, k, out_stride, true));
  if (tokens == 0) return PSKV_OK;
  if ((n_rows && !rows) || !place || !out) return set_error(PSKV_EINVAL, "null buffer");
  const size_t size = type_bytes(type);
  const RowSpan to{out, tokens, k, out_stride, size};
  const uint64_t listed = tokens * choices * 4;
  if (rows_overlap({rows, n_rows, k, rows_stride, size}, to) || rows_overlap(stretch(place, listed), to) ||
      rows_overlap(stretch(weights, listed), to))
    return set_error(PSKV_EINVAL, "the rows that are written overlap what is read");
  DeviceGuard guard(device);
  if (!guard.ok()) return set_error(PSKV_EHIP, "cannot select device %d", device);
  // (without rows there is no row 0 to read either)
  const RowArgs a = row_args(tokens, n_rows ? choices : 0, n_rows, k, out_stride, rows_stride, type, lanes_of(tokens));
  with_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    with_flag((1 + choices) * tokens * k * size > kPastBytes, [&](auto far) {
      constexpr bool PAST = decltype(far)::value;
      auto kernel = a.lanes_log2 >= 6 ? k_route_sum<T, true, PAST> : k_route_sum<T, false, PAST>;
      hipLaunchKernelGGL(kernel, dim3(a.groups), dim3(kRowBlock), 0,
                         static_cast<hipStream_t>(stream), static_cast<const T*>(rows), place, weights, static_cast<T*>(out), a);
    });
  });
  PSKV_HIP(hipGetLastError());
  return PSKV_OK;
}

extern "C" int pskv_route_sum_grad(int device, void* stream, int type, const void* grad, size_t grad_stride, size_t tokens,
                                   size_t k, const void* rows, size_t rows_stride, size_t n_rows, const int32_t* place,
                                   const float* weights, size_t choices, void* grad_rows, size_t grad_rows_stride,
                                   float* grad_weights) {
  clear_error();
  RETURN_IF(check_rows(type, tokens, choices, n_rows, k));
  RETURN_IF(check_stride("grad", tokens, k, grad_stride, false));
  RETURN_IF(check_stride("rows", n_rows, k, rows_stride, false));
  RETURN_IF(check_stride("grad_rows", n_rows, k, grad_rows_stride, true));
  if (tokens == 0) return PSKV_OK;
  if (!grad || !place || !weights || !grad_weights || (n_rows && (!rows || !grad_rows)))
    return set_error(PSKV_EINVAL, "null buffer");
  const size_t size = type_bytes(type);
  const uint64_t listed = tokens * choices * 4;
  const RowSpan to{grad_rows, n_rows, k, grad_rows_stride, size}, to_weights = stretch(grad_weights, listed);
  if (rows_overlap(to, to_weights)) return set_error(PSKV_EINVAL, "the gradients of the rows and of the weights overlap");
  for (const RowSpan& read : {RowSpan{grad, tokens, k, grad_stride, size}, RowSpan{rows, n_rows, k, rows_stride, size},
                              stretch(place, listed), stretch(weights, listed)})
    if (rows_overlap(read, to) || rows_overlap(read, to_weights))
      return set_error(PSKV_EINVAL, "the gradients that are written overlap what is read");
  DeviceGuard guard(device);
  if (!guard.ok()) return set_error(PSKV_EHIP, "cannot select device %d", device);
  RowArgs a = row_args(tokens, choices, n_rows, k, grad_stride, rows_stride, type, 64);
  // (300 tokens x 8 choices of 1,024 bf16: all of a token in one wavefront 14.2 us, in eight 5.6)
  unsigned share = (unsigned)choices;
  while (share > 1 && ((tokens * ((choices + share - 1) / share)) << a.lanes_log2) < 64 * 4096) share = (share + 1) / 2;
  a.groups = grid_for(tokens * ((choices + share - 1) / share), kRowBlock >> a.lanes_log2, 1u << 22);
  with_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    with_flag((1 + 2 * choices) * tokens * k * size > kPastBytes, [&](auto far) {
      constexpr bool PAST = decltype(far)::value;
      const uint64_t vectors = k / Row<T>::kWide;
      auto kernel = a.lanes_log2 < 6     ? k_route_sum_grad<T, false, PAST, 1, false>
                    : vectors <= 64      ? k_route_sum_grad<T, true, PAST, 1, false>
                    : vectors <= 128     ? k_route_sum_grad<T, true, PAST, 2, false>
                    : vectors <= 4 * 64 ? k_route_sum_grad<T, true, PAST, 4, false>
                                         : k_route_sum_grad<T, true, PAST, 4, true>;
      hipLaunchKernelGGL(kernel, dim3(a.groups), dim3(kRowBlock), 0,
                         static_cast<hipStream_t>(stream), static_cast<const T*>(grad), static_cast<const T*>(rows), place, weights,
                         static_cast<T*>(grad_rows), (uint64_t)grad_rows_stride, grad_weights, share, a);
    });
  });
  PSKV_HIP(hipGetLastError());
  return PSKV_OK;
}
