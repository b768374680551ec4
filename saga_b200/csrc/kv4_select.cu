// Block selection: scores of the complete pages from their key bounds, then the
// `top` best per (request, key head).
//
// For a page with per-channel bounds lo <= k <= hi, q.k <= sum_d q_d * (q_d > 0
// ? hi_d : lo_d). Products and sums are binary32 with a fixed tree (halves:
// d with d + D/2, then d + D/4, ...), so the scores, and with them the
// selection, do not depend on how the work is laid out.
#include <algorithm>

#include "kv4.cuh"

namespace saga {

namespace {

constexpr int kTopThreads = 512;
constexpr int kTopKeys = 8192;  // keys kept in shared memory; further ones are made again from the scores

// Order-preserving key of a score: NaN lowest, -0 as +0; 0 is below every score.
__device__ __forceinline__ uint32_t score_key(float x) {
  if (x != x) return 1u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Sums v[0..NV-1] over the warp, value by value in the same tree as a butterfly
// from distance 16 down to 1, halving the live values at each step: lane l ends
// with the sum of value l / (32 / NV).
template <int NV>
__device__ __forceinline__ float warp_sums(float (&v)[NV]) {
  const int lane = threadIdx.x & 31;
  int o = 16;
#pragma unroll
  for (int n = NV / 2; n > 0; n >>= 1, o >>= 1) {
    const bool up = (lane & o) != 0;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float send = up ? v[i] : v[i + n];
      v[i] = __fadd_rn(up ? v[i + n] : v[i], __shfl_xor_sync(0xffffffffu, send, o));
    }
  }
#pragma unroll
  for (; o > 0; o >>= 1) v[0] = __fadd_rn(v[0], __shfl_xor_sync(0xffffffffu, v[0], o));
  return v[0];
}

// A warp scores one page at a time for the heads of one key head, NV at a time
// in registers: lane l has channels l, l + 32 (l + 64, l + 96), so the first
// levels of the tree are its own and the last five go across the warp.
template <typename T, int D, int NV>
__global__ void __launch_bounds__(256) kv4_score_kernel(SagaKv4Args a, float* __restrict__ scores) {
  constexpr int N = D / 32;
  pdl_wait();
  const int G = a.Hq / a.pool.Hk;
  const int row = blockIdx.y;
  const int b = row / a.pool.Hk, kh = row % a.pool.Hk;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int pl = a.pool.page_len;
  const int len = min(max(a.lens[b], 0), a.max_pages * pl);
  const int pages = (len + pl - 1) / pl;
  if (pages <= a.top) return;  // all are kept
  const int step = gridDim.x * (blockDim.x >> 5);
  // the kept pages at either end need no score
  const int j0 = a.keep_first + blockIdx.x * (blockDim.x >> 5) + warp, j1 = pages - a.keep_last;
  if (j0 >= j1) return;
  const T* q = reinterpret_cast<const T*>(a.q) + (int64_t)b * a.q_sb + (int64_t)kh * G * a.q_sh;
  for (int g0 = 0; g0 < G; g0 += NV) {
    float qv[NV][N];
#pragma unroll
    for (int g = 0; g < NV; ++g)
#pragma unroll
      for (int i = 0; i < N; ++i)
        qv[g][i] = g0 + g < G ? Num<T>::to_f(q[(int64_t)(g0 + g) * a.q_sh + lane + 32 * i]) : 0.f;
    // pages of this warp: lane i finds the i-th of the next 32
    for (int base = j0; base < j1; base += 32 * step) {
      int mine = 0;
      if (base + lane * step < j1) {
        mine = a.page_table[(int64_t)b * a.pt_sb + base + lane * step];
        if (mine < 0 || mine >= a.pool.num_pages) {
          set_status(a.status, SAGA_STATUS_PAGE_RANGE);
          mine = 0;
        }
      }
      const int n = min(32, (j1 - base + step - 1) / step);
      __nv_bfloat16 lo[N], hi[N];
      auto fetch = [&](int x) {
        const int page = __shfl_sync(0xffffffffu, mine, x);
        const int64_t at = ((int64_t)page * a.pool.Hk + kh) * D + lane;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          lo[i] = reinterpret_cast<const __nv_bfloat16*>(a.pool.k_lo)[at + 32 * i];
          hi[i] = reinterpret_cast<const __nv_bfloat16*>(a.pool.k_hi)[at + 32 * i];
        }
      };
      fetch(0);
      for (int x = 0; x < n; ++x) {
        float l[N], h[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          l[i] = __bfloat162float(lo[i]);
          h[i] = __bfloat162float(hi[i]);
        }
        if (x + 1 < n) fetch(x + 1);
        float s[NV];
#pragma unroll
        for (int g = 0; g < NV; ++g) {
          float y[N];
#pragma unroll
          for (int i = 0; i < N; ++i) y[i] = __fmul_rn(qv[g][i], qv[g][i] > 0.f ? h[i] : l[i]);
#pragma unroll
          for (int m = N / 2; m > 0; m >>= 1)
#pragma unroll
            for (int i = 0; i < m; ++i) y[i] = __fadd_rn(y[i], y[i + m]);
          s[g] = y[0];
        }
        float best = warp_sums<NV>(s);
        if (g0 + lane / (32 / NV) >= G) best = -INFINITY;
        best = warp_nanmax(best);
        if (lane == 0) {
          float* to = scores + (int64_t)row * a.max_pages + base + x * step;
          *to = g0 == 0 ? best : nanmax(*to, best);
        }
      }
    }
  }
}

// One CTA per (request, key head): the key of the top-th best page by four
// passes over 8 bits of the keys, then the pages above it and the lowest pages
// at it, in ascending order.
__global__ void __launch_bounds__(kTopThreads) kv4_top_kernel(SagaKv4Args a, const float* __restrict__ scores) {
  __shared__ int hist[256];
  __shared__ int sh_bin, sh_left;
  __shared__ int wsum[2][kTopThreads / 32];
  __shared__ uint32_t keys[kTopKeys];
  pdl_wait();
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
  auto make_key = [&](int j) -> uint32_t {
    return (j < a.keep_first || j >= pages - a.keep_last) ? 0xffffffffu : score_key(s[j]);
  };
  for (int j = threadIdx.x; j < min(pages, kTopKeys); j += kTopThreads) keys[j] = make_key(j);
  auto key_of = [&](int j) -> uint32_t { return j < kTopKeys ? keys[j] : make_key(j); };
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
  const int G = a.Hq / a.pool.Hk;
  if (rows > 65535) return abi_fail(SAGA_ERR_UNSUPPORTED, "more than 65535 (request, key head) rows");
  if (a.max_pages > a.top) {
    // a page per warp until every SM has eight CTAs
    const int want = (a.max_pages + 7) / 8, most = std::max(1, 8 * 148 / rows);
    const dim3 grid(std::min(want, most), rows);
    auto go = [&](auto* t, auto d) {
      using T = std::remove_pointer_t<decltype(t)>;
      return kv4_launch("kv4_score_kernel",
                        G <= 4   ? kv4_score_kernel<T, d.value, 4>
                        : G <= 8 ? kv4_score_kernel<T, d.value, 8>
                                 : kv4_score_kernel<T, d.value, 16>,
                        grid, 256, 0, st, a, scores);
    };
    auto by_d = [&](auto* t) {
      return a.pool.D == 128 ? go(t, std::integral_constant<int, 128>()) : go(t, std::integral_constant<int, 64>());
    };
    const int rc = a.dtype == SAGA_BF16   ? by_d((__nv_bfloat16*)nullptr)
                   : a.dtype == SAGA_FP16 ? by_d((__half*)nullptr)
                                          : by_d((float*)nullptr);
    if (rc) return rc;
  }
  return kv4_launch("kv4_top_kernel", kv4_top_kernel, dim3(rows), kTopThreads, 0, st, a, scores);
}

}  // namespace saga
