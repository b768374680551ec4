// Quantised writes into the 4-bit paged cache, reads of what it stands for, and
// the key bounds of completed pages.
#include <algorithm>
#include <type_traits>

#include "kv4.cuh"

namespace saga {

namespace {

// Two lanes hold one group, every second 16 bytes of its values each, so that
// loads and stores take whole sectors; they exchange codes so that each leaves
// (or reads) one of the group's two 16-byte chunks. What is done once per group (the
// address, the scale) costs as much as ten values, so fewer lanes with more values
// each are cheaper: 131,072 tokens of five heads of 128 in bf16 (215 MB) are written
// in 98 us by eight lanes, 51 us by four (whose schedulers issue in 83 % of the cycles)
// and 39.5 us by two, 5.4 TB/s; read in 39.6 us by four and 36.4 us by two, 5.9 TB/s.
// The rows go past the caches (__ldcs, __stcs): a prompt's rows are larger than L2, and
// the read took 3 us more without. CTAs of 256 threads write the same in 43.4 us, of 64 in 40.
constexpr int kLanes = 2;
constexpr int kVals = 64 / kLanes;
constexpr int kCtaThreads = 128;
constexpr int kCtaGroups = kCtaThreads / kLanes;
constexpr int kAhead = 2;  // groups that a lane loads before it works on the first

// A lane's values as they are loaded: every second 16 bytes of the group.
template <typename T>
struct Raw {
  uint4 w[kVals * sizeof(T) / 16];
};
template <typename T>
constexpr int kPiece = 16 / sizeof(T);  // values of one load
template <typename T, bool VEC>
__device__ __forceinline__ void load_vals(const T* p, Raw<T>& r) {
#pragma unroll
  for (int h = 0; h < kVals / kPiece<T>; ++h) {
    if constexpr (VEC) {
      r.w[h] = __ldcs(reinterpret_cast<const uint4*>(p + kLanes * kPiece<T> * h));
    } else {
#pragma unroll
      for (int i = 0; i < kPiece<T>; ++i) reinterpret_cast<T*>(&r.w[h])[i] = p[kLanes * kPiece<T> * h + i];
    }
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_vals(T* p, const Raw<T>& r) {
#pragma unroll
  for (int h = 0; h < kVals / kPiece<T>; ++h) {
    if constexpr (VEC) {
      __stcs(reinterpret_cast<uint4*>(p + kLanes * kPiece<T> * h), r.w[h]);
    } else {
#pragma unroll
      for (int i = 0; i < kPiece<T>; ++i) p[kLanes * kPiece<T> * h + i] = reinterpret_cast<const T*>(&r.w[h])[i];
    }
  }
}

// Least and greatest of a lane's values, and a value that is not 0 if
// one of them is NaN or infinite. The 16-bit types are compared in pairs.
template <typename T>
__device__ __forceinline__ void extremes(const Raw<T>& r, float& lo, float& hi, float& odd) {
  if constexpr (sizeof(T) == 4) {
    const float* x = reinterpret_cast<const float*>(&r);
    lo = hi = x[0];
    odd = x[0] * 0.f;
#pragma unroll
    for (int i = 1; i < kVals; ++i) {
      lo = fminf(lo, x[i]);
      hi = fmaxf(hi, x[i]);
      odd = fmaf(x[i], 0.f, odd);
    }
  } else {
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    const T2* x = reinterpret_cast<const T2*>(&r);
    T2 zero;
    *reinterpret_cast<uint32_t*>(&zero) = 0u;
    T2 a = x[0], b = x[0], o = __hmul2(x[0], zero);
#pragma unroll
    for (int i = 1; i < kVals / 2; ++i) {
      a = __hmin2(a, x[i]);
      b = __hmax2(b, x[i]);
      o = __hfma2(x[i], zero, o);
    }
    lo = fminf(Num<T>::to_f(a.x), Num<T>::to_f(a.y));
    hi = fmaxf(Num<T>::to_f(b.x), Num<T>::to_f(b.y));
    odd = Num<T>::to_f(o.x) + Num<T>::to_f(o.y);
  }
}

struct Rows {  // keys or values, [T, H, D]
  int64_t st, sh;
  uint8_t* pool;
  int H;
};

// How the groups of T tokens are dealt out: a CTA has `strip` tokens, all heads
// and groups of each; `magic` divides by the groups of a token.
struct Deal {
  int64_t T;
  int strip, per;
  uint32_t magic;
  int tpp_shift;   // log2 of the tiles per page
  int64_t slots;   // of the pool
};

// Unit u of the CTA's strip: its values, and the tile of its slot if that is in
// the pool.
template <int D>
struct Unit {
  uint8_t* tile;  // NULL: no slot
  int64_t src;    // element offset of the lane's values in the tensor
  int row, g;
  bool is_v;
  bool live;  // the token exists
};
template <int D, int PIECE>
__device__ __forceinline__ Unit<D> locate_unit(uint32_t u, const Deal& d, const Rows& kr, const Rows& vr,
                                               const int64_t* __restrict__ slots, int l, int* status) {
  constexpr int NG = D / 64;
  Unit<D> x;
  const uint32_t tl = __umulhi(u, d.magic);  // u / per
  const int rest = (int)(u - tl * (uint32_t)d.per);
  const int64_t t = (int64_t)blockIdx.x * d.strip + tl;
  x.live = (int)tl < d.strip && t < d.T;
  const int64_t slot = x.live ? slots[t] : -1;
  x.g = rest % NG;
  int h = rest / NG;
  x.is_v = h >= kr.H;
  if (x.is_v) h -= kr.H;
  x.src = t * (x.is_v ? vr.st : kr.st) + h * (x.is_v ? vr.sh : kr.sh) + x.g * 64 + l * PIECE;
  const bool inside = slot >= 0 && slot < d.slots;
  if (!inside && slot != -1 && rest == 0 && l == 0) set_status(status, SAGA_STATUS_PAGE_RANGE);
  x.row = (int)slot & (kKv4Tile - 1);
  const uint32_t ptile = (uint32_t)(slot / kKv4Tile);  // the host checks that the pool's tiles fit an int
  const uint32_t page = ptile >> d.tpp_shift, in_page = ptile & ((1u << d.tpp_shift) - 1u);
  const int64_t tile = (((int64_t)page * (x.is_v ? vr.H : kr.H) + h) << d.tpp_shift) + in_page;
  x.tile = inside ? (x.is_v ? vr.pool : kr.pool) + tile * kv4_tile_bytes(D) : nullptr;
  return x;
}
// w[h]: the codes of a lane's values 8h .. 8h + 7. In the tile lane l has chunk l,
// so the two lanes exchange what the other needs. 16-bit types: w[h] is word 2h + l
// of the group. fp32: its halves are those of words 2h and 2h + 1, the lower ones
// in lane 0, the upper ones in lane 1.
template <typename T>
__device__ __forceinline__ uint4 chunk_of_codes(const uint32_t (&w)[4], int l) {
  const uint32_t r0 = __shfl_xor_sync(0xffffffffu, l ? w[0] : w[2], 1);
  const uint32_t r1 = __shfl_xor_sync(0xffffffffu, l ? w[1] : w[3], 1);
  if constexpr (sizeof(T) == 2) return l ? make_uint4(r0, w[2], r1, w[3]) : make_uint4(w[0], r0, w[1], r1);
  const uint32_t a0 = l ? r0 : w[0], a1 = l ? r1 : w[1], b0 = l ? w[2] : r0, b1 = l ? w[3] : r1;
  return make_uint4(__byte_perm(a0, b0, 0x5410), __byte_perm(a0, b0, 0x7632), __byte_perm(a1, b1, 0x5410),
                    __byte_perm(a1, b1, 0x7632));
}
template <typename T>
__device__ __forceinline__ void codes_of_chunk(const uint4& c, int l, uint32_t (&w)[4]) {
  uint32_t even[2] = {c.x, c.z}, odd[2] = {c.y, c.w};  // words of lane 0 and of lane 1
  if constexpr (sizeof(T) == 4) {
    even[0] = __byte_perm(c.x, c.y, 0x5410);
    even[1] = __byte_perm(c.z, c.w, 0x5410);
    odd[0] = __byte_perm(c.x, c.y, 0x7632);
    odd[1] = __byte_perm(c.z, c.w, 0x7632);
  }
  const uint32_t r0 = __shfl_xor_sync(0xffffffffu, l ? even[0] : odd[0], 1);
  const uint32_t r1 = __shfl_xor_sync(0xffffffffu, l ? even[1] : odd[1], 1);
  w[0] = l ? r0 : even[0];
  w[1] = l ? r1 : even[1];
  w[2] = l ? odd[0] : r0;
  w[3] = l ? odd[1] : r1;
}
template <int D>
__device__ __forceinline__ uint4* chunk_at(const Unit<D>& x, int l) {
  return reinterpret_cast<uint4*>(x.tile + kv4_chunk_off<D>(x.row, x.g * 2 + l));
}

constexpr float kMagic = 8388608.f;  // 2^23: adding it rounds to a whole number, to nearest even

template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(kCtaThreads) kv4_write_kernel(const T* __restrict__ k, const T* __restrict__ v,
                                                                Rows kr, Rows vr, Deal deal,
                                                                const int64_t* __restrict__ slots, int* status) {
  constexpr int AHEAD = sizeof(T) == 4 ? 1 : kAhead;  // fp32: 32 registers a group
  // (65,536 tokens of five heads of 128: 30.7 us, 32.1 us with two)
  pdl_wait();
  const int l = threadIdx.x & (kLanes - 1);
  const uint32_t units = (uint32_t)deal.strip * (uint32_t)deal.per;
  const unsigned lanes = 3u << (threadIdx.x & 30);
  for (uint32_t u0 = 0; u0 < units; u0 += kCtaGroups * AHEAD) {  // the same trips for all lanes of a warp
    Unit<D> at[AHEAD];
    Raw<T> raw[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      at[i] = locate_unit<D, kPiece<T>>(u0 + i * kCtaGroups + threadIdx.x / kLanes, deal, kr, vr, slots, l, status);
      raw[i] = Raw<T>();
      if (at[i].tile) load_vals<T, VEC>((at[i].is_v ? v : k) + at[i].src, raw[i]);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      float lo, hi, odd;
      extremes<T>(raw[i], lo, hi, odd);
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      }
      // rounded down and up, so that z and z + 15 s enclose the group
      const __nv_bfloat16 zb = bf16_down(lo);
      const float z = __bfloat162float(zb);
      const __nv_bfloat16 sb = bf16_up(fmaxf(__fmul_rn(__fsub_rn(hi, z), 1.0f / 15.0f), 0x1p-40f));
      const float s = __bfloat162float(sb);
      const bool bad = (__ballot_sync(0xffffffffu, odd != 0.f) & lanes) != 0 || !isfinite(z) || !isfinite(s);
      const float inv = __frcp_rn(s);
      // (x - z) / s lies in [0, 15] but for its rounding, so the nearest whole number is a code without
      // a clamp. It is rounded by adding 2^23; the words 0x4b000000 + code are summed at their places
      // and what the constants amount to is taken off.
      const f32x2 minus_z = pack2(-z, -z);
      constexpr uint32_t kOff = 0x4b000000u + (0x4b000000u << 4);  // the higher places overflow
      const T* x = reinterpret_cast<const T*>(&raw[i]);
      uint32_t w[4];
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        w[h] = 0;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          float y0, y1;
          unpack2(add2(pack2(Num<T>::to_f(x[8 * h + j]), Num<T>::to_f(x[8 * h + j + 1])), minus_z), y0, y1);
          // not packed: the assembler joins a packed product with the packed sum after it
          w[h] += __float_as_uint(__fadd_rn(__fmul_rn(y0, inv), kMagic)) << (4 * j);
          w[h] += __float_as_uint(__fadd_rn(__fmul_rn(y1, inv), kMagic)) << (4 * j + 4);
        }
        w[h] = bad ? 0u : w[h] - kOff;
      }
      const uint4 c = chunk_of_codes<T>(w, l);
      if (at[i].tile) *chunk_at<D>(at[i], l) = c;
      if (l == 0 && at[i].tile) {
        const uint32_t m = (uint32_t)__bfloat16_as_ushort(sb) | ((uint32_t)__bfloat16_as_ushort(zb) << 16);
        // s = 0 and z = NaN for a group that is not finite: whatever the codes are, it stands for NaN, and the
        // greatest scale of a row, which places the weights of the attention, is that of its other group
        *reinterpret_cast<uint32_t*>(at[i].tile + kv4_meta_off<D>(at[i].row, at[i].g)) = bad ? 0x7fff0000u : m;
      }
    }
  }
}

// The eight codes of a word as pairs of binary32 values: y[j] has codes j and j + 4.
// Put into the low bits of the fp16 number 1024, a code (or 16 times a code) is
// exact; in that form two take one logical and one fp16 instruction.
__device__ __forceinline__ void codes8(uint32_t w, f32x2 (&y)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t u = (j < 2 ? w : w >> 8) & (j & 1 ? 0x00f000f0u : 0x000f000fu) | 0x64006400u;
    const __half2 one = __floats2half2_rn(j & 1 ? 0.0625f : 1.f, j & 1 ? 0.0625f : 1.f);
    const __half2 off = __floats2half2_rn(j & 1 ? -64.f : -1024.f, j & 1 ? -64.f : -1024.f);
    const float2 c = __half22float2(__hfma2(*reinterpret_cast<const __half2*>(&u), one, off));
    y[j] = pack2(c.x, c.y);
  }
}

template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(kCtaThreads) kv4_read_kernel(T* __restrict__ k, T* __restrict__ v, Rows kr, Rows vr,
                                                               Deal deal, const int64_t* __restrict__ slots,
                                                               int* status) {
  pdl_wait();
  const int l = threadIdx.x & (kLanes - 1);
  const uint32_t units = (uint32_t)deal.strip * (uint32_t)deal.per;
  for (uint32_t u0 = 0; u0 < units; u0 += kCtaGroups * kAhead) {
    Unit<D> at[kAhead];
    uint4 c[kAhead];
    uint32_t m[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      at[i] = locate_unit<D, kPiece<T>>(u0 + i * kCtaGroups + threadIdx.x / kLanes, deal, kr, vr, slots, l, status);
      c[i] = make_uint4(0u, 0u, 0u, 0u);
      m[i] = 0u;
      if (at[i].tile) {
        c[i] = *chunk_at<D>(at[i], l);
        m[i] = *reinterpret_cast<const uint32_t*>(at[i].tile + kv4_meta_off<D>(at[i].row, at[i].g));
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      uint32_t w[4];
      codes_of_chunk<T>(c[i], l, w);
      if (!at[i].live) continue;
      const float s = kv4_scale(m[i]), z = kv4_zero(m[i]);
      Raw<T> r;
      T* x = reinterpret_cast<T*>(&r);
      const f32x2 s2 = pack2(s, s), z2 = pack2(z, z);
      // s * code has at most 12 significant bits, so the sum is rounded once
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        f32x2 y[4];
        codes8(w[h], y);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float y0, y1;
          unpack2(fma2(s2, y[j], z2), y0, y1);
          x[8 * h + j] = Num<T>::from_f(y0);
          x[8 * h + j + 4] = Num<T>::from_f(y1);
        }
      }
      store_vals<T, VEC>((at[i].is_v ? v : k) + at[i].src, r);
    }
  }
}

// Bounds of the pages whose last slot is among the slots: a CTA looks at
// `strip` tokens and takes the bounds of the pages that they complete. Threads
// split a page into D/8 words of a row by 16 (32) rows. 1024 pages of 128 rows of
// 128 take 10 us after the write that completes them (one page at a time and its
// loads' latency: the schedulers issue in a third of the cycles); four rows of a
// thread on their way together, since eight need 80 registers and leave fewer
// CTAs per SM (13 us).
constexpr int kBoundThreads = 256;
template <int D>
__global__ void __launch_bounds__(kBoundThreads) kv4_bounds_kernel(SagaKv4Pool p, int64_t T_, int strip,
                                                         const int64_t* __restrict__ slots) {
  constexpr int W = D / 8, ROWS = kBoundThreads / W;
  __shared__ __align__(16) float red[2][ROWS][D];
  __shared__ int64_t done[kBoundThreads];
  __shared__ int n_done;
  if (threadIdx.x == 0) n_done = 0;
  pdl_wait();
  __syncthreads();
  const int w = threadIdx.x % W, rr = threadIdx.x / W;
  const int64_t t = (int64_t)blockIdx.x * strip + threadIdx.x;
  const int64_t slot = (int)threadIdx.x < strip && t < T_ ? slots[t] : -1;
  if (slot >= 0 && slot < (int64_t)p.num_pages * p.page_len && (slot & (p.page_len - 1)) == p.page_len - 1)
    done[atomicAdd(&n_done, 1)] = slot / p.page_len;  // in any order: each page is by itself
  __syncthreads();
  const int n = n_done;
  for (int x = 0; x < n; ++x) {
    const int64_t page = done[x];
    for (int h = 0; h < p.Hk; ++h) {
      float lo[8], hi[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        lo[i] = INFINITY;
        hi[i] = -INFINITY;
      }
#pragma unroll 4
      for (int off = rr; off < p.page_len; off += ROWS) {
        const uint8_t* tile =
            reinterpret_cast<const uint8_t*>(p.k) + kv4_tile_at<D>(page, h, p.Hk, off, p.page_len);
        const int row = off % kKv4Tile;
        const uint32_t c =
            *reinterpret_cast<const uint32_t*>(tile + kv4_chunk_off<D>(row, w >> 2) + (w & 3) * 4);
        const uint32_t m = *reinterpret_cast<const uint32_t*>(tile + kv4_meta_off<D>(row, w >> 3));
        const float s = kv4_scale(m), z = kv4_zero(m);
        const f32x2 s2 = pack2(s, s), z2 = pack2(z, z);
        f32x2 y[4];
        codes8(c, y);
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // NaN rows are left out (fminf and fmaxf return the other operand)
          float x0, x1;
          unpack2(fma2(s2, y[j], z2), x0, x1);
          lo[j] = fminf(lo[j], x0);
          hi[j] = fmaxf(hi[j], x0);
          lo[j + 4] = fminf(lo[j + 4], x1);
          hi[j + 4] = fmaxf(hi[j + 4], x1);
        }
      }
#pragma unroll
      for (int i = 0; i < 8; i += 4) {  // the word's fourths of all words together: no bank conflicts
        *reinterpret_cast<float4*>(&red[0][rr][i * W + 4 * w]) = make_float4(lo[i], lo[i + 1], lo[i + 2], lo[i + 3]);
        *reinterpret_cast<float4*>(&red[1][rr][i * W + 4 * w]) = make_float4(hi[i], hi[i + 1], hi[i + 2], hi[i + 3]);
      }
      __syncthreads();
      if (threadIdx.x < D) {
        float a = red[0][0][threadIdx.x], b = red[1][0][threadIdx.x];
#pragma unroll
        for (int i = 1; i < ROWS; ++i) {
          a = fminf(a, red[0][i][threadIdx.x]);
          b = fmaxf(b, red[1][i][threadIdx.x]);
        }
        if (a > b) a = b = __int_as_float(0x7fffffff);  // no key stands for a number here
        const int d = (int)threadIdx.x % (4 * W) / 4 * 8 + (int)threadIdx.x / (4 * W) * 4 + (int)threadIdx.x % 4;
        const int64_t at = (page * p.Hk + h) * D + d;
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

// A CTA's strip is cut so that its groups fill all lanes kAhead deep, or to one
// token where there are too few tokens to fill the SMs so.
static int make_deal(const SagaKv4Pool& p, int64_t T, Deal* d, unsigned* grid) {
  d->T = T;
  d->per = (p.Hk + p.Hv) * (p.D / 64);
  const int full = std::max(1, kAhead * kCtaGroups / d->per);
  d->strip = (int)std::max<int64_t>(1, std::min<int64_t>(full, T / (2 * sm_count())));
  // exact for u * per < 2^32; u stays below strip * per + 2 kAhead kCtaGroups
  d->magic = (uint32_t)(((1ull << 32) + d->per - 1) / d->per);
  if ((uint64_t)((int64_t)d->strip * d->per + 2 * kAhead * kCtaGroups) * d->per >= (1ull << 32) || d->per < 2)
    return abi_fail(SAGA_ERR_UNSUPPORTED, "too many heads");
  d->tpp_shift = 0;
  while ((kKv4Tile << d->tpp_shift) < p.page_len) ++d->tpp_shift;
  d->slots = (int64_t)p.num_pages * p.page_len;
  const int64_t n = (T + d->strip - 1) / d->strip;
  if (n > 0x7fffffffll) return abi_fail(SAGA_ERR_UNSUPPORTED, "too many rows for one call");
  *grid = (unsigned)n;
  return SAGA_OK;
}

int launch_kv4_write(const SagaKv4Pool& p, int dt, int64_t T, const void* k, int64_t k_st, int64_t k_sh,
                     const void* v, int64_t v_st, int64_t v_sh, const int64_t* slots, int* status, cudaStream_t st) {
  const int esz = dt == SAGA_FP32 ? 4 : 2;
  const bool vec = rows_aligned(k, k_st, k_sh, esz) && rows_aligned(v, v_st, v_sh, esz);
  const Rows kr{k_st, k_sh, reinterpret_cast<uint8_t*>(p.k), p.Hk};
  const Rows vr{v_st, v_sh, reinterpret_cast<uint8_t*>(p.v), p.Hv};
  Deal deal;
  unsigned grid;
  int rc = make_deal(p, T, &deal, &grid);
  if (rc) return rc;
  dispatch(dt, p.D, vec, [&](auto* t, auto d, auto a) {
    using E = std::remove_pointer_t<decltype(t)>;
    rc = kv4_launch("kv4_write_kernel", kv4_write_kernel<E, d.value, a.value>, dim3(grid), kCtaThreads, 0, st,
                    reinterpret_cast<const E*>(k), reinterpret_cast<const E*>(v), kr, vr, deal, slots, status);
  });
  if (rc || !p.k_lo) return rc;
  // One token per CTA where every token may complete a page, as the tokens of that many requests can (4096 of
  // them 29 us, by strips 450 us); a run of prompt tokens completes one in page_len (4096 of them 8 us with a
  // CTA each, 5 us by strips; from 1024 down the same).
  const int strip = T <= 4096 ? 1 : std::min(p.page_len, kBoundThreads);
  const unsigned nb = (unsigned)((T + strip - 1) / strip);
  return kv4_launch("kv4_bounds_kernel", p.D == 128 ? kv4_bounds_kernel<128> : kv4_bounds_kernel<64>, dim3(nb),
                    kBoundThreads, 0, st, p, T, strip, slots);
}

int launch_kv4_read(const SagaKv4Pool& p, int dt, int64_t T, const int64_t* slots, void* k, int64_t k_st,
                    int64_t k_sh, void* v, int64_t v_st, int64_t v_sh, int* status, cudaStream_t st) {
  const int esz = dt == SAGA_FP32 ? 4 : 2;
  const bool vec = rows_aligned(k, k_st, k_sh, esz) && rows_aligned(v, v_st, v_sh, esz);
  const Rows kr{k_st, k_sh, reinterpret_cast<uint8_t*>(p.k), p.Hk};
  const Rows vr{v_st, v_sh, reinterpret_cast<uint8_t*>(p.v), p.Hv};
  Deal deal;
  unsigned grid;
  int rc = make_deal(p, T, &deal, &grid);
  if (rc) return rc;
  dispatch(dt, p.D, vec, [&](auto* t, auto d, auto a) {
    using E = std::remove_pointer_t<decltype(t)>;
    rc = kv4_launch("kv4_read_kernel", kv4_read_kernel<E, d.value, a.value>, dim3(grid), kCtaThreads, 0, st,
                    reinterpret_cast<E*>(k), reinterpret_cast<E*>(v), kr, vr, deal, slots, status);
  });
  return rc;
}

}  // namespace saga
