// Quantised writes into the 4-bit paged cache, reads of what it stands for, and
// the key bounds of completed pages.
#include "kv4.cuh"

namespace saga {

namespace {

// Eight lanes hold one group: lane l has its values 8l .. 8l + 7, so a row's
// 16-bit values arrive in 16-byte loads and leave as one word of codes per lane,
// 32 consecutive bytes (one sector) per group.
constexpr int kLanesPerGroup = 8;

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, float* f) {
  if constexpr (VEC) {
    load8f<T>(p, f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = Num<T>::to_f(p[i]);
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, const float* f) {
  T t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = Num<T>::from_f(f[i]);
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
      reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(t)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = t[i];
  }
}

struct Rows {  // keys or values, [T, H, D]
  int64_t st, sh;
  uint8_t* pool;
  int H;
};

// The group of eight lanes that the calling thread belongs to handles unit u:
// token u / (H * NG), head and group from the rest.
template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(256) kv4_write_kernel(const T* __restrict__ k, const T* __restrict__ v, Rows kr,
                                                        Rows vr, int64_t T_, const int64_t* __restrict__ slots,
                                                        int page_len, int num_pages, int* status) {
  pdl_wait();
  constexpr int NG = D / 64;
  const int l = threadIdx.x & (kLanesPerGroup - 1);
  const int64_t u = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / kLanesPerGroup;
  const int per = (kr.H + vr.H) * NG;
  const int64_t t = u / per;
  // lanes past the end keep taking part in the shuffles below
  int64_t slot = t < T_ ? slots[t] : -1;
  const int rest = (int)(u - t * per);
  const int g = rest % NG;
  int h = rest / NG;
  if (slot < 0 || slot >= (int64_t)num_pages * page_len) {
    if (slot != -1 && rest == 0 && l == 0) set_status(status, SAGA_STATUS_PAGE_RANGE);
    slot = -1;
  }
  const bool is_v = h >= kr.H;
  if (is_v) h -= kr.H;
  const Rows r = is_v ? vr : kr;
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = 0.f;
  if (slot >= 0) load8<T, VEC>((is_v ? v : k) + t * r.st + h * r.sh + g * 64 + l * 8, x);
  float lo = x[0], hi = x[0];
  bool bad = !isfinite(x[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    bad |= !isfinite(x[i]);
  }
#pragma unroll
  for (int o = kLanesPerGroup / 2; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const unsigned lanes = 0xffu << (threadIdx.x & 24);
  bad = (__ballot_sync(0xffffffffu, bad) & lanes) != 0;
  // rounded down and up, so that z and z + 15 s enclose the group
  const __nv_bfloat16 zb = bf16_down(lo);
  const float z = __bfloat162float(zb);
  const __nv_bfloat16 sb = bf16_up(fmaxf(__fmul_rn(__fsub_rn(hi, z), 1.0f / 15.0f), 0x1p-40f));
  const float s = __bfloat162float(sb);
  bad = bad || !isfinite(z) || !isfinite(s);
  const float inv = __frcp_rn(s);
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(x[i], z), inv)), 0.f), 15.f);
    w |= (uint32_t)c << (4 * i);
  }
  if (slot < 0) return;
  const int off = (int)(slot & (page_len - 1));
  uint8_t* tile = r.pool + kv4_tile_at<D>(slot / page_len, h, r.H, off, page_len);
  const int row = off % kKv4Tile;
  *reinterpret_cast<uint32_t*>(tile + kv4_chunk_off<D>(row, g * 2 + (l >> 2)) + (l & 3) * 4) = bad ? 0u : w;
  if (l == 0) {
    const uint32_t m = (uint32_t)__bfloat16_as_ushort(sb) | ((uint32_t)__bfloat16_as_ushort(zb) << 16);
    *reinterpret_cast<uint32_t*>(tile + kv4_meta_off<D>(row, g)) = bad ? 0x7fff7fffu : m;
  }
}

template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(256) kv4_read_kernel(T* __restrict__ k, T* __restrict__ v, Rows kr, Rows vr,
                                                       int64_t T_, const int64_t* __restrict__ slots, int page_len,
                                                       int num_pages, int* status) {
  pdl_wait();
  constexpr int NG = D / 64;
  const int l = threadIdx.x & (kLanesPerGroup - 1);
  const int64_t u = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / kLanesPerGroup;
  const int per = (kr.H + vr.H) * NG;
  const int64_t t = u / per;
  if (t >= T_) return;
  const int64_t slot = slots[t];
  const int rest = (int)(u - t * per);
  const int g = rest % NG;
  int h = rest / NG;
  const bool is_v = h >= kr.H;
  if (is_v) h -= kr.H;
  const Rows r = is_v ? vr : kr;
  float x[8];
  if (slot < 0 || slot >= (int64_t)num_pages * page_len) {
    if (slot != -1 && rest == 0 && l == 0) set_status(status, SAGA_STATUS_PAGE_RANGE);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
  } else {
    const int off = (int)(slot & (page_len - 1));
    const uint8_t* tile = r.pool + kv4_tile_at<D>(slot / page_len, h, r.H, off, page_len);
    const int row = off % kKv4Tile;
    const uint32_t w =
        *reinterpret_cast<const uint32_t*>(tile + kv4_chunk_off<D>(row, g * 2 + (l >> 2)) + (l & 3) * 4);
    const uint32_t m = *reinterpret_cast<const uint32_t*>(tile + kv4_meta_off<D>(row, g));
    const float s = kv4_scale(m), z = kv4_zero(m);
    // s * code has at most 12 significant bits, so the sum is rounded once
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __fmaf_rn(s, (float)((w >> (4 * i)) & 15u), z);
  }
  store8<T, VEC>((is_v ? v : k) + t * r.st + h * r.sh + g * 64 + l * 8, x);
}

// Bounds of the pages whose last slot is among the slots: a CTA looks at
// `strip` tokens and takes the bounds of the pages that they complete. Threads
// split a page into D/8 words of a row by 8 (16) rows.
template <int D>
__global__ void __launch_bounds__(128) kv4_bounds_kernel(SagaKv4Pool p, int64_t T_, int strip,
                                                         const int64_t* __restrict__ slots) {
  constexpr int W = D / 8, ROWS = 128 / W;
  __shared__ float red[2][ROWS][D];
  pdl_wait();
  const int w = threadIdx.x % W, rr = threadIdx.x / W;
  for (int64_t t = (int64_t)blockIdx.x * strip; t < min((int64_t)(blockIdx.x + 1) * strip, T_); ++t) {
    const int64_t slot = slots[t];
    if (slot < 0 || slot >= (int64_t)p.num_pages * p.page_len || (slot & (p.page_len - 1)) != p.page_len - 1)
      continue;
    const int64_t page = slot / p.page_len;
    for (int h = 0; h < p.Hk; ++h) {
      float lo[8], hi[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        lo[i] = INFINITY;
        hi[i] = -INFINITY;
      }
      for (int off = rr; off < p.page_len; off += ROWS) {
        const uint8_t* tile =
            reinterpret_cast<const uint8_t*>(p.k) + kv4_tile_at<D>(page, h, p.Hk, off, p.page_len);
        const int row = off % kKv4Tile;
        const uint32_t c =
            *reinterpret_cast<const uint32_t*>(tile + kv4_chunk_off<D>(row, w >> 2) + (w & 3) * 4);
        const uint32_t m = *reinterpret_cast<const uint32_t*>(tile + kv4_meta_off<D>(row, w >> 3));
        const float s = kv4_scale(m), z = kv4_zero(m);
#pragma unroll
        for (int i = 0; i < 8; ++i) {  // NaN rows are left out (fminf and fmaxf return the other operand)
          const float x = __fmaf_rn(s, (float)((c >> (4 * i)) & 15u), z);
          lo[i] = fminf(lo[i], x);
          hi[i] = fmaxf(hi[i], x);
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        red[0][rr][w * 8 + i] = lo[i];
        red[1][rr][w * 8 + i] = hi[i];
      }
      __syncthreads();
      if (threadIdx.x < D) {
        float a = red[0][0][threadIdx.x], b = red[1][0][threadIdx.x];
#pragma unroll
        for (int i = 1; i < ROWS; ++i) {
          a = fminf(a, red[0][i][threadIdx.x]);
          b = fmaxf(b, red[1][i][threadIdx.x]);
        }
        const int64_t at = (page * p.Hk + h) * D + threadIdx.x;
        reinterpret_cast<__nv_bfloat16*>(p.k_lo)[at] = bf16_down(a);
        reinterpret_cast<__nv_bfloat16*>(p.k_hi)[at] = bf16_up(b);
      }
      __syncthreads();
    }
  }
}

bool rows_aligned(const void* p, int64_t st, int64_t sh, int esz) {
  return (reinterpret_cast<uintptr_t>(p) % 16) == 0 && (st * esz) % 16 == 0 && (sh * esz) % 16 == 0;
}

// Calls f with a null pointer of the element type, D and the alignment as
// compile-time constants.
template <class F>
void dispatch(int dt, int D, bool vec, F f) {
  auto by_vec = [&](auto* t, auto d) {
    if (vec) f(t, d, std::true_type());
    else f(t, d, std::false_type());
  };
  auto by_d = [&](auto* t) {
    if (D == 128) by_vec(t, std::integral_constant<int, 128>());
    else by_vec(t, std::integral_constant<int, 64>());
  };
  if (dt == SAGA_BF16) by_d((__nv_bfloat16*)nullptr);
  else if (dt == SAGA_FP16) by_d((__half*)nullptr);
  else by_d((float*)nullptr);
}

}  // namespace

int launch_kv4_write(const SagaKv4Pool& p, int dt, int64_t T, const void* k, int64_t k_st, int64_t k_sh,
                     const void* v, int64_t v_st, int64_t v_sh, const int64_t* slots, int* status, cudaStream_t st) {
  const int esz = dt == SAGA_FP32 ? 4 : 2;
  const bool vec = rows_aligned(k, k_st, k_sh, esz) && rows_aligned(v, v_st, v_sh, esz);
  const Rows kr{k_st, k_sh, reinterpret_cast<uint8_t*>(p.k), p.Hk};
  const Rows vr{v_st, v_sh, reinterpret_cast<uint8_t*>(p.v), p.Hv};
  const int64_t threads = T * (p.Hk + p.Hv) * (p.D / 64) * kLanesPerGroup;
  const int64_t grid = (threads + 255) / 256;
  if (grid > 0x7fffffffll) return abi_fail(SAGA_ERR_UNSUPPORTED, "too many rows for one call");
  int rc = SAGA_OK;
  dispatch(dt, p.D, vec, [&](auto* t, auto d, auto a) {
    using E = std::remove_pointer_t<decltype(t)>;
    rc = kv4_launch("kv4_write_kernel", kv4_write_kernel<E, d.value, a.value>, dim3((unsigned)grid), 256, 0, st,
                    reinterpret_cast<const E*>(k), reinterpret_cast<const E*>(v), kr, vr, T, slots, p.page_len,
                    p.num_pages, status);
  });
  if (rc || !p.k_lo) return rc;
  const int strip = T <= 4096 ? 1 : 32;
  const unsigned nb = (unsigned)((T + strip - 1) / strip);
  return kv4_launch("kv4_bounds_kernel", p.D == 128 ? kv4_bounds_kernel<128> : kv4_bounds_kernel<64>, dim3(nb), 128, 0,
                    st, p, T, strip, slots);
}

int launch_kv4_read(const SagaKv4Pool& p, int dt, int64_t T, const int64_t* slots, void* k, int64_t k_st,
                    int64_t k_sh, void* v, int64_t v_st, int64_t v_sh, int* status, cudaStream_t st) {
  const int esz = dt == SAGA_FP32 ? 4 : 2;
  const bool vec = rows_aligned(k, k_st, k_sh, esz) && rows_aligned(v, v_st, v_sh, esz);
  const Rows kr{k_st, k_sh, reinterpret_cast<uint8_t*>(p.k), p.Hk};
  const Rows vr{v_st, v_sh, reinterpret_cast<uint8_t*>(p.v), p.Hv};
  const int64_t threads = T * (p.Hk + p.Hv) * (p.D / 64) * kLanesPerGroup;
  const int64_t grid = (threads + 255) / 256;
  if (grid > 0x7fffffffll) return abi_fail(SAGA_ERR_UNSUPPORTED, "too many rows for one call");
  int rc = SAGA_OK;
  dispatch(dt, p.D, vec, [&](auto* t, auto d, auto a) {
    using E = std::remove_pointer_t<decltype(t)>;
    rc = kv4_launch("kv4_read_kernel", kv4_read_kernel<E, d.value, a.value>, dim3((unsigned)grid), 256, 0, st,
                    reinterpret_cast<E*>(k), reinterpret_cast<E*>(v), kr, vr, T, slots, p.page_len, p.num_pages,
                    status);
  });
  return rc;
}

}  // namespace saga
