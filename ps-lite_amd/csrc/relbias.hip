// The learned relative position bias and its gradient (gfx950):
//     out[b,h,i,j] = scores[b,h,i,j] + table[bucket(rel)][h],  rel = (k_first + j) - (q_first + q_at[b] + i)
//     dtable[u][h] = sum of grad[b,h,i,j] over the b, i, j whose bucket is u
// The bias depends on j - i alone, so a tile of R rows and C columns needs R + C - 1 values of it, which are worked out once
// and kept in LDS; the gradient sums diagonals first, a lane to each, and diagonals into buckets once per workgroup.
#include <hip/hip_runtime.h>

#include <new>

#include "host_common.h"
#include "relbias.h"
#include "row_types.h"

namespace pskv {
namespace {

constexpr unsigned kBlock = 256;
constexpr unsigned kCols = 1024, kRows = 32;  // a tile of the bias

struct Shape {
  uint64_t B, H, Q, K;
  int64_t rel0;  // of row 0, column 0, before q_at
  uint64_t in[3], out[3];  // strides of batch, head and row
};

template <typename T, bool SCORES>
__global__ __launch_bounds__(kBlock) void k_relbias(const float* __restrict__ table, const int64_t* __restrict__ q_at,
                                                     const T* scores, T* out, Shape s, Buckets b) {
  __shared__ float bias[kRows + kCols];
  const uint64_t c0 = (uint64_t)blockIdx.x * kCols, r0 = (uint64_t)blockIdx.y * kRows;
  const unsigned cols = s.K - c0 < kCols ? (unsigned)(s.K - c0) : kCols;
  const unsigned rows = s.Q - r0 < kRows ? (unsigned)(s.Q - r0) : kRows;
  for (uint64_t z = blockIdx.z; z < s.B * s.H; z += gridDim.z) {
    const uint64_t batch = z / s.H, head = z % s.H;
    // bias[x]: of the diagonal x - (rows - 1) of the tile
    const uint64_t rel = (uint64_t)s.rel0 - (q_at ? (uint64_t)q_at[batch] : 0) + c0 - r0 - (rows - 1);
    __syncthreads();
    for (unsigned x = threadIdx.x; x < rows + cols - 1; x += kBlock)
      bias[x] = table[(uint64_t)bucket_of(b, (int64_t)(rel + x)) * s.H + head];
    __syncthreads();
    const T* from = SCORES ? scores + batch * s.in[0] + head * s.in[1] + r0 * s.in[2] + c0 : nullptr;
    T* to = out + batch * s.out[0] + head * s.out[1] + r0 * s.out[2] + c0;
    for (unsigned i = 0; i < rows; ++i)
      for (unsigned j = threadIdx.x; j < cols; j += kBlock) {
        const float v = bias[j + rows - 1 - i];
        to[i * s.out[2] + j] = (T)(SCORES ? (float)from[i * s.in[2] + j] + v : v);
      }
  }
}

// --- the gradient ------------------------------------------------------------------------------------------------

constexpr unsigned kSumRows = 128;  // rows of a strip

// A strip: kSumRows rows of one head (of all batches, or of one where they are at positions of their own). A workgroup takes 256
// neighbouring diagonals of it, a lane adds up one diagonal, row by row and batch by batch.
// partial[head][bucket][workgroup of the head].
template <typename T>
__global__ __launch_bounds__(kBlock) void k_relbias_sums(const T* __restrict__ grad, const int64_t* __restrict__ q_at,
                                                          float* __restrict__ partial, unsigned buckets, unsigned slots,
                                                          unsigned strips, Shape s, Buckets b) {
  __shared__ float acc[kBlock / 64][kMostBuckets];
  const uint64_t head = blockIdx.z;
  const unsigned strip = blockIdx.y % strips;
  const uint64_t batch0 = q_at ? blockIdx.y / strips : 0, batches = q_at ? 1 : s.B;
  const uint64_t r0 = (uint64_t)strip * kSumRows;
  const unsigned rows = s.Q - r0 < kSumRows ? (unsigned)(s.Q - r0) : kSumRows;
  const unsigned wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (unsigned u = lane; u < buckets; u += 64) acc[wave][u] = 0.0f;
  __syncthreads();
  // column = diag + row within the strip
  const int64_t diag = (int64_t)((uint64_t)blockIdx.x * kBlock + threadIdx.x) - (int64_t)(rows - 1);
  float sum = 0.0f;
  for (uint64_t n = 0; n < batches; ++n) {
    const T* from = grad + (batch0 + n) * s.in[0] + head * s.in[1] + r0 * s.in[2];
    float mine = 0.0f;
#pragma unroll 8
    for (unsigned i = 0; i < rows; ++i) {
      const int64_t j = diag + i;
      if (j >= 0 && j < (int64_t)s.K) mine += (float)from[i * s.in[2] + j];
    }
    sum += mine;
  }
  const uint64_t rel = (uint64_t)s.rel0 - (q_at ? (uint64_t)q_at[batch0] : 0) + (uint64_t)diag - r0;
  const unsigned u = diag < (int64_t)s.K ? bucket_of(b, (int64_t)rel) : kMostBuckets;
  // lanes of one bucket are neighbours: a sum over each stretch of them, left at its last lane
  unsigned start = __shfl_up(u, 1) != u || lane == 0 ? lane : 0;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned up = __shfl_up(start, o);
    if (lane >= (unsigned)o && up > start) start = up;
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const float up = __shfl_up(sum, o);
    if (lane >= start + o) sum += up;
  }
  const unsigned next = __shfl_down(u, 1);
  if (u < buckets && (lane == 63 || next != u)) acc[wave][u] = sum;
  __syncthreads();
  const unsigned slot = blockIdx.y * gridDim.x + blockIdx.x;
  for (unsigned v = threadIdx.x; v < buckets; v += kBlock) {
    float t = acc[0][v];
#pragma unroll
    for (unsigned w = 1; w < kBlock / 64; ++w) t += acc[w][v];
    partial[(head * buckets + v) * slots + slot] = t;
  }
}

__global__ __launch_bounds__(kBlock) void k_relbias_join(const float* __restrict__ partial, unsigned buckets, unsigned slots,
                                                          uint64_t H, float* __restrict__ grad_table) {
  __shared__ float red[kBlock / 64];
  const uint64_t head = blockIdx.y;
  const unsigned u = blockIdx.x;
  const float* from = partial + (head * buckets + u) * slots;
  float sum = 0.0f;
  for (unsigned i = threadIdx.x; i < slots; i += kBlock) sum += from[i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    float t = red[0];
    for (unsigned w = 1; w < kBlock / 64; ++w) t += red[w];
    grad_table[(uint64_t)u * H + head] = t;
  }
}

// --- the host's checks -------------------------------------------------------------------------------------------

int check(int type, size_t H, size_t B, size_t Q, size_t K, int64_t q_first, int64_t k_first) {
  if (!type_bytes(type)) return set_error(PSKV_EINVAL, "type %d: PSKV_F32, PSKV_F16 or PSKV_BF16", type);
  if (H == 0 || H > 65535) return set_error(PSKV_EINVAL, "1 to 65535 heads");
  if (B > (1u << 20) || Q > (1u << 20) || K > (1u << 30)) return set_error(PSKV_EINVAL, "sizes beyond what one call handles");
  const int64_t most = 1ll << 60;
  if (q_first > most || q_first < -most || k_first > most || k_first < -most)
    return set_error(PSKV_EINVAL, "positions beyond 2^60");
  return PSKV_OK;
}

int buckets_or_error(Buckets* b, size_t buckets, uint64_t max_distance, int two_sided) {
  bool ok = false;
  try {
    ok = make_buckets(b, buckets, max_distance, two_sided != 0);
  } catch (const std::bad_alloc&) {
    return set_error(PSKV_ENOMEM, "no memory for the borders of the buckets");
  }
  if (!ok)
    return set_error(PSKV_EINVAL, "%zu buckets up to distance %llu: 2 (two-sided 4) to %u buckets, and a distance beyond those with "
                     "a bucket of their own, up to 2^30", buckets, (unsigned long long)max_distance, kMostBuckets);
  return PSKV_OK;
}

// The bytes from the first element of a [B, H, Q, K] tensor to behind its last.
uint64_t extent(const int64_t* stride, const Shape& s, size_t size) {
  return ((s.B - 1) * (uint64_t)stride[0] + (s.H - 1) * (uint64_t)stride[1] + (s.Q - 1) * (uint64_t)stride[2] + s.K) * size;
}

int check_strides(const char* what, const int64_t* stride, const Shape& s, bool written) {
  if (!stride) return set_error(PSKV_EINVAL, "%s: no strides", what);
  uint64_t n[4] = {s.B, s.H, s.Q, s.K}, by[4] = {(uint64_t)stride[0], (uint64_t)stride[1], (uint64_t)stride[2], 1};
  for (int i = 0; i < 3; ++i)
    if (stride[i] < 0 || stride[i] > (1ll << 40)) return set_error(PSKV_EINVAL, "%s: strides of 0 to 2^40", what);
  if (!written) return PSKV_OK;
  // every element has a place of its own: the next wider stride begins behind what the narrower ones reach
  for (int i = 0; i < 4; ++i)
    for (int j = i + 1; j < 4; ++j)
      if (by[j] < by[i] || (by[j] == by[i] && n[j] < n[i])) {
        const uint64_t x = by[i], y = n[i];
        by[i] = by[j], n[i] = n[j];
        by[j] = x, n[j] = y;
      }
  uint64_t reach = 0;
  for (int i = 0; i < 4; ++i) {
    if (n[i] < 2) continue;
    if (by[i] <= reach) return set_error(PSKV_EINVAL, "%s: elements that are written lie upon each other", what);
    reach += (n[i] - 1) * by[i];
  }
  return PSKV_OK;
}

struct SumPlan {
  unsigned across, strips, down, slots;
  SumPlan(size_t B, size_t Q, size_t K, bool own_positions) {
    const size_t rows = Q < kSumRows ? Q : kSumRows;
    across = (unsigned)((K + rows - 1 + kBlock - 1) / kBlock);
    strips = (unsigned)((Q + kSumRows - 1) / kSumRows);
    down = strips * (unsigned)(own_positions ? B : 1);
    slots = across * down;
  }
};

}  // namespace
}  // namespace pskv

using namespace pskv;

static_assert(kMostBuckets == PSKV_RELBIAS_MAX_BUCKETS, "the header says so");

extern "C" int pskv_relbias_bucket(int64_t rel, size_t buckets, uint64_t max_distance, int two_sided) {
  clear_error();
  Buckets b;
  const int rc = buckets_or_error(&b, buckets, max_distance, two_sided);
  return rc ? rc : (int)bucket_of(b, rel);
}

extern "C" int pskv_relbias(int device, void* stream, int type, const float* table, size_t buckets, size_t H,
                            uint64_t max_distance, int two_sided, int64_t q_first, int64_t k_first, const int64_t* q_at,
                            const void* scores, const int64_t* scores_stride, void* out, const int64_t* out_stride, size_t B,
                            size_t Q, size_t K) {
  clear_error();
  int rc = check(type, H, B, Q, K, q_first, k_first);
  if (rc) return rc;
  Buckets b;
  if ((rc = buckets_or_error(&b, buckets, max_distance, two_sided))) return rc;
  if (B == 0 || Q == 0 || K == 0) return PSKV_OK;
  if (!table || !out) return set_error(PSKV_EINVAL, "null buffer");
  Shape s{B, H, Q, K, k_first - q_first, {0, 0, 0}, {0, 0, 0}};
  if ((rc = check_strides("out", out_stride, s, true))) return rc;
  if (scores && (rc = check_strides("scores", scores_stride, s, false))) return rc;
  for (int i = 0; i < 3; ++i) {
    s.out[i] = (uint64_t)out_stride[i];
    s.in[i] = scores ? (uint64_t)scores_stride[i] : 0;
  }
  if (scores) {
    const uint64_t a = reinterpret_cast<uintptr_t>(scores), o = reinterpret_cast<uintptr_t>(out), size = type_bytes(type);
    bool same = a == o;
    const size_t n[3] = {B, H, Q};
    for (int i = 0; i < 3; ++i) same = same && (n[i] < 2 || s.in[i] == s.out[i]);
    if (!same && a < o + extent(out_stride, s, size) && o < a + extent(scores_stride, s, size))
      return set_error(PSKV_EINVAL, "out lies in the scores and is not the same tensor");
  }
  DeviceGuard guard(device);
  if (!guard.ok()) return set_error(PSKV_EHIP, "cannot select device %d", device);
  const dim3 grid((unsigned)((K + kCols - 1) / kCols), (unsigned)((Q + kRows - 1) / kRows),
                  (unsigned)(B * H < 65535 ? B * H : 65535));
  with_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    auto kernel = scores ? k_relbias<T, true> : k_relbias<T, false>;
    hipLaunchKernelGGL(kernel, grid, dim3(kBlock), 0, static_cast<hipStream_t>(stream), table, q_at,
                       static_cast<const T*>(scores), static_cast<T*>(out), s, b);
  });
  PSKV_HIP(hipGetLastError());
  return PSKV_OK;
}

extern "C" size_t pskv_relbias_grad_room(size_t buckets, size_t H, size_t B, size_t Q, size_t K, int own_positions) {
  if (B == 0 || Q == 0 || K == 0 || B > (1u << 20) || Q > (1u << 20) || K > (1u << 30)) return 0;
  return SumPlan(B, Q, K, own_positions != 0).slots * buckets * H * sizeof(float);
}

extern "C" int pskv_relbias_grad(int device, void* stream, int type, const void* grad, const int64_t* grad_stride,
                                 size_t buckets, size_t H, uint64_t max_distance, int two_sided, int64_t q_first,
                                 int64_t k_first, const int64_t* q_at, size_t B, size_t Q, size_t K, float* grad_table,
                                 void* work, size_t work_bytes) {
  clear_error();
  int rc = check(type, H, B, Q, K, q_first, k_first);
  if (rc) return rc;
  Buckets b;
  if ((rc = buckets_or_error(&b, buckets, max_distance, two_sided))) return rc;
  if (!grad_table) return set_error(PSKV_EINVAL, "null buffer");
  Shape s{B, H, Q, K, k_first - q_first, {0, 0, 0}, {0, 0, 0}};
  SumPlan plan(B, Q, K, q_at != nullptr);
  const bool any = B && Q && K;
  if (any) {
    if (!grad) return set_error(PSKV_EINVAL, "null buffer");
    if ((rc = check_strides("grad", grad_stride, s, false))) return rc;
    for (int i = 0; i < 3; ++i) s.in[i] = (uint64_t)grad_stride[i];
    const size_t room = pskv_relbias_grad_room(buckets, H, B, Q, K, q_at != nullptr);
    if (!work || work_bytes < room || (reinterpret_cast<uintptr_t>(work) & 3))
      return set_error(PSKV_EINVAL, "this gradient takes %zu bytes of working memory, %zu given", room, work ? work_bytes : (size_t)0);
    if (plan.down > 65535) return set_error(PSKV_EINVAL, "sizes beyond what one call handles");
  }
  DeviceGuard guard(device);
  if (!guard.ok()) return set_error(PSKV_EHIP, "cannot select device %d", device);
  hipStream_t st = static_cast<hipStream_t>(stream);
  float* partial = static_cast<float*>(work);
  if (any)
    with_type(type, [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      hipLaunchKernelGGL(k_relbias_sums<T>, dim3(plan.across, plan.down, (unsigned)H), dim3(kBlock), 0, st,
                         static_cast<const T*>(grad), q_at, partial, (unsigned)buckets, plan.slots, plan.strips, s, b);
    });
  hipLaunchKernelGGL(k_relbias_join, dim3((unsigned)buckets, (unsigned)H), dim3(kBlock), 0, st, partial, (unsigned)buckets,
                     any ? plan.slots : 0u, (uint64_t)H, grad_table);
  PSKV_HIP(hipGetLastError());
  return PSKV_OK;
}
