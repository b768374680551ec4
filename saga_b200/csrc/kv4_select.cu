// Block selection: scores of the complete pages from their key bounds, then the
// `top` best per (request, key head).
//
// For a page with per-channel bounds lo <= k <= hi, q.k <= sum_d q_d * (q_d > 0
// ? hi_d : lo_d). Products and sums are binary32 with a fixed tree (halves:
// d with d + D/2, then d + D/4, ...), so the scores, and with them the
// selection, do not depend on how the work is laid out.
#include "kv4.cuh"

namespace saga {

namespace {

constexpr int kTopThreads = 256;

// Order-preserving key of a score: NaN lowest, -0 as +0; 0 is below every score.
__device__ __forceinline__ uint32_t score_key(float x) {
  if (x != x) return 1u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// A warp scores one page at a time for all heads of one key head: lane l has
// channels l, l + 32 (l + 64, l + 96), so the first levels of the tree are its
// own and the last five are a butterfly.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_score_kernel(SagaKv4Args a, float* __restrict__ scores) {
  constexpr int N = D / 32;
  extern __shared__ float qs[];  // [G][D]
  const int G = a.Hq / a.pool.Hk;
  const int row = blockIdx.y;
  const int b = row / a.pool.Hk, kh = row % a.pool.Hk;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int pl = a.pool.page_len;
  const int len = min(max(a.lens[b], 0), a.max_pages * pl);
  const int pages = (len + pl - 1) / pl;
  if (pages <= a.top) return;  // all are kept
  const T* q = reinterpret_cast<const T*>(a.q) + (int64_t)b * a.q_sb + (int64_t)kh * G * a.q_sh;
  for (int i = threadIdx.x; i < G * D; i += blockDim.x) qs[i] = Num<T>::to_f(q[(int64_t)(i / D) * a.q_sh + i % D]);
  __syncthreads();
  const int step = gridDim.x * (blockDim.x >> 5);
  // the kept pages at either end need no score
  for (int j = a.keep_first + blockIdx.x * (blockDim.x >> 5) + warp; j < pages - a.keep_last; j += step) {
    int page = a.page_table[(int64_t)b * a.pt_sb + j];
    if (page < 0 || page >= a.pool.num_pages) {
      if (lane == 0) set_status(a.status, SAGA_STATUS_PAGE_RANGE);
      page = 0;
    }
    const int64_t at = ((int64_t)page * a.pool.Hk + kh) * D;
    float lo[N], hi[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      lo[i] = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.pool.k_lo)[at + lane + 32 * i]);
      hi[i] = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.pool.k_hi)[at + lane + 32 * i]);
    }
    float best = -INFINITY;
    for (int g = 0; g < G; ++g) {
      float x[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float qv = qs[g * D + lane + 32 * i];
        x[i] = __fmul_rn(qv, qv > 0.f ? hi[i] : lo[i]);
      }
#pragma unroll
      for (int n = N / 2; n > 0; n >>= 1)
#pragma unroll
        for (int i = 0; i < n; ++i) x[i] = __fadd_rn(x[i], x[i + n]);
      float s = x[0];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s = __fadd_rn(s, __shfl_xor_sync(0xffffffffu, s, o));
      best = nanmax(best, s);
    }
    if (lane == 0) scores[(int64_t)row * a.max_pages + j] = best;
  }
}

// One CTA per (request, key head): the key of the top-th best page by four
// passes over 8 bits of the keys, then the pages above it and the lowest pages
// at it, in ascending order.
__global__ void __launch_bounds__(kTopThreads) kv4_top_kernel(SagaKv4Args a, const float* __restrict__ scores) {
  __shared__ int hist[256];
  __shared__ int sh_bin, sh_left;
  __shared__ int wsum[2][kTopThreads / 32];
  const int row = blockIdx.x;
  const int b = row / a.pool.Hk;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int pl = a.pool.page_len;
  if (a.lens[b] > a.max_pages * pl && threadIdx.x == 0) set_status(a.status, SAGA_STATUS_PAGE_RANGE);
  const int len = min(max(a.lens[b], 0), a.max_pages * pl);
  const int pages = (len + pl - 1) / pl;
  int32_t* out = a.blocks + (int64_t)row * a.top;
  if (threadIdx.x == 0) a.counts[row] = min(pages, a.top);
  if (pages <= a.top) {
    for (int i = threadIdx.x; i < a.top; i += kTopThreads) out[i] = i < pages ? i : -1;
    return;
  }
  const float* s = scores + (int64_t)row * a.max_pages;
  auto key_of = [&](int j) -> uint32_t {
    return (j < a.keep_first || j >= pages - a.keep_last) ? 0xffffffffu : score_key(s[j]);
  };
  uint32_t prefix = 0;
  int left = a.top;  // pages still to take among those that match the prefix
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += kTopThreads) hist[i] = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < pages; j += kTopThreads) {
      const uint32_t k = key_of(j);
      if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255u], 1);
    }
    __syncthreads();
    if (warp == 0) {  // the bin that holds the left-th greatest: lane l has bins 255 - 8l .. 248 - 8l
      int c[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += (c[i] = hist[255 - 8 * lane - i]);
      int above = warp_incl_scan(sum) - sum;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (above < left && left <= above + c[i]) {
          sh_bin = 255 - 8 * lane - i;
          sh_left = left - above;
        }
        above += c[i];
      }
    }
    __syncthreads();
    prefix |= (uint32_t)sh_bin << shift;
    left = sh_left;
  }
  int done_gt = 0, done_eq = 0;  // pages above the key and at it so far
  for (int base = 0; base < pages; base += kTopThreads) {
    const int j = base + threadIdx.x;
    const uint32_t k = j < pages ? key_of(j) : 0u;
    const bool gt = k > prefix, eq = j < pages && k == prefix;
    const unsigned bg = __ballot_sync(0xffffffffu, gt), be = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) {
      wsum[0][warp] = __popc(bg);
      wsum[1][warp] = __popc(be);
    }
    __syncthreads();
    int g = done_gt, e = done_eq;
#pragma unroll
    for (int w = 0; w < kTopThreads / 32; ++w) {
      if (w < warp) {
        g += wsum[0][w];
        e += wsum[1][w];
      }
      done_gt += wsum[0][w];
      done_eq += wsum[1][w];
    }
    const unsigned below = (1u << lane) - 1u;
    g += __popc(bg & below);
    e += __popc(be & below);
    if (gt || (eq && e < left)) out[g + min(e, left)] = j;
    __syncthreads();
  }
}

}  // namespace

size_t kv4_select_workspace(const SagaKv4Args& a) {
  return ((size_t)a.B * a.pool.Hk * a.max_pages * sizeof(float) + 255) / 256 * 256 + 256;
}

int launch_kv4_select(const SagaKv4Args& a, cudaStream_t st) {
  float* scores = reinterpret_cast<float*>(a.workspace);
  const int rows = a.B * a.pool.Hk;
  const int smem = a.Hq / a.pool.Hk * a.pool.D * (int)sizeof(float);
  if (smem > 48 * 1024) return abi_fail(SAGA_ERR_UNSUPPORTED, "too many query heads per key head");
  if (rows > 65535) return abi_fail(SAGA_ERR_UNSUPPORTED, "more than 65535 (request, key head) rows");
  if (a.max_pages > a.top) {
    const dim3 grid((a.max_pages + 63) / 64, rows);
    auto go = [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      if (a.pool.D == 128) kv4_score_kernel<T, 128><<<grid, 256, smem, st>>>(a, scores);
      else kv4_score_kernel<T, 64><<<grid, 256, smem, st>>>(a, scores);
    };
    if (a.dtype == SAGA_BF16) go((__nv_bfloat16*)nullptr);
    else if (a.dtype == SAGA_FP16) go((__half*)nullptr);
    else go((float*)nullptr);
    if (int rc = kv4_launched("kv4_score_kernel")) return rc;
  }
  kv4_top_kernel<<<rows, kTopThreads, 0, st>>>(a, scores);
  return kv4_launched("kv4_top_kernel");
}

}  // namespace saga
