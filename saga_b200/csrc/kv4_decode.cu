// Attention of one query position per request over the 4-bit paged cache.
#include "kv4.cuh"

namespace saga {

namespace {

// One CTA per (request, query head); each warp takes every eighth position, a
// lane has D/32 channels, with a running maximum and sum per warp.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) kv4_decode_simple_kernel(SagaKv4Args a) {
  constexpr int N = D / 32;  // channels of a lane: N consecutive ones
  __shared__ float sm_m[kWarps], sm_l[kWarps], sm_o[kWarps][D];
  const int b = blockIdx.x / a.Hq, h = blockIdx.x % a.Hq;
  const int kh = h / (a.Hq / a.pool.Hk), vh = h / (a.Hq / a.pool.Hv);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int pl = a.pool.page_len;
  if (a.lens[b] > a.max_pages * pl && threadIdx.x == 0) set_status(a.status, SAGA_STATUS_PAGE_RANGE);
  const int len = min(max(a.lens[b], 0), a.max_pages * pl);
  const int start = a.starts ? max(a.starts[b], 0) : 0;
  const int32_t* blocks = a.blocks ? a.blocks + ((int64_t)b * a.pool.Hk + kh) * a.top : nullptr;
  const int n = blocks ? min(max(a.counts[b * a.pool.Hk + kh], 0), a.top) * pl : len;
  const T* q = reinterpret_cast<const T*>(a.q) + (int64_t)b * a.q_sb + (int64_t)h * a.q_sh + lane * N;
  float qv[N], o[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    qv[i] = Num<T>::to_f(q[i]) * a.scaling;
    o[i] = 0.f;
  }
  const int g = lane * N / 64;
  auto load = [&](const void* pool, int64_t page, int head, int H, int off, float* x) {
    const uint8_t* tile = reinterpret_cast<const uint8_t*>(pool) + kv4_tile_at<D>(page, head, H, off, pl);
    const int row = off % kKv4Tile, by = lane * N / 2;
    const uint8_t* c = tile + kv4_chunk_off<D>(row, by >> 4) + (by & 15);
    const uint32_t m = *reinterpret_cast<const uint32_t*>(tile + kv4_meta_off<D>(row, g));
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = __fmaf_rn(kv4_scale(m), (float)((c[i / 2] >> (4 * (i & 1))) & 15), kv4_zero(m));
  };
  float m = -INFINITY, l = 0.f;
  for (int i = warp; i < n; i += kWarps) {
    int pi = i / pl;
    if (blocks) {
      pi = blocks[pi];
      if (pi < 0 || pi >= a.max_pages) continue;
    }
    const int pos = pi * pl + i % pl;
    if (pos < start || pos >= len) continue;
    int page = a.page_table[(int64_t)b * a.pt_sb + pi];
    if (page < 0 || page >= a.pool.num_pages) {
      if (lane == 0) set_status(a.status, SAGA_STATUS_PAGE_RANGE);
      page = 0;
    }
    float x[N], s = 0.f;
    load(a.pool.k, page, kh, a.pool.Hk, i % pl, x);
#pragma unroll
    for (int j = 0; j < N; ++j) s = fmaf(qv[j], x[j], s);
    s = warp_sum(s);
    const float mn = fmaxf(m, s);
    const float f = m == -INFINITY ? 0.f : __expf(m - mn);
    const float p = mn == -INFINITY ? 0.f : expf(s - mn);
    load(a.pool.v, page, vh, a.pool.Hv, i % pl, x);
    l = l * f + p;
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = o[j] * f + p * x[j];
    m = mn;
  }
  if (lane == 0) {
    sm_m[warp] = m;
    sm_l[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) sm_o[warp][lane * N + i] = o[i];
  __syncthreads();
  if (threadIdx.x < D) {
    float M = -INFINITY, L = 0.f, O = 0.f;
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm_m[w]);
    for (int w = 0; w < kWarps; ++w) {
      const float f = sm_m[w] == -INFINITY ? 0.f : expf(sm_m[w] - M);
      L += sm_l[w] * f;
      O += sm_o[w][threadIdx.x] * f;
    }
    reinterpret_cast<T*>(a.out)[(int64_t)b * a.o_sb + (int64_t)h * a.o_sh + threadIdx.x] =
        Num<T>::from_f(L > 0.f || L != L ? O / L : 0.f);
  }
}

}  // namespace

size_t kv4_decode_workspace(const SagaKv4Args& a) { return 256; }

int launch_kv4_decode(const SagaKv4Args& a, cudaStream_t st) {
  const unsigned grid = (unsigned)(a.B * a.Hq);
  auto go = [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (a.pool.D == 128) kv4_decode_simple_kernel<T, 128><<<grid, kThreads, 0, st>>>(a);
    else kv4_decode_simple_kernel<T, 64><<<grid, kThreads, 0, st>>>(a);
  };
  if (a.dtype == SAGA_BF16) go((__nv_bfloat16*)nullptr);
  else if (a.dtype == SAGA_FP16) go((__half*)nullptr);
  else go((float*)nullptr);
  return kv4_launched("kv4_decode_simple_kernel");
}

}  // namespace saga
