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
constexpr int kTopKeys = 8192;  // keys kept in shared memory; further ones are read again

// Order-preserving key of a score, -0 as +0; kNanKey is below every number's and 0 below that.
constexpr uint32_t kNanKey = 1u;
__device__ __forceinline__ uint32_t score_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Sums v[0..3] over the warp, each in the same tree as a butterfly from distance
// 16 down to 1, halving the live values at the first two steps: lane l ends with
// the sum of value l / 8.
__device__ __forceinline__ float warp_sums4(float (&v)[4]) {
  const int lane = threadIdx.x & 31;
  bool up = (lane & 16) != 0;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    v[i] = __fadd_rn(up ? v[i + 2] : v[i], __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i + 2], 16));
  up = (lane & 8) != 0;
  float s = __fadd_rn(up ? v[1] : v[0], __shfl_xor_sync(0xffffffffu, up ? v[0] : v[1], 8));
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) s = __fadd_rn(s, __shfl_xor_sync(0xffffffffu, s, o));
  return s;
}

constexpr int kScoreBatch = 2;  // pages whose bounds a warp loads together
constexpr int kScorePages = 8;  // pages per warp, at most (a multiple of the batch)

// A warp scores `per_warp` consecutive pages for the heads of one key head, 4 NC
// of them at a time in registers: lane l has channels l, l + 32 (l + 64, l + 96),
// so the first levels of the tree are its own and the last five go across the
// warp. Scores are written as keys. 23,400 pages of 64 rows (ragged contexts of up
// to 65,600 in pages of 64), 12 heads of 128, take 20 us for 12 MB of bounds: 33
// instructions per page and head, issued in half of the cycles, over 1.2 waves of
// CTAs. Shorter runs than eight pages per warp wait more often for their first
// loads, longer ones leave SMs idle (4: 27.6 us with the choice of the pages, 8:
// 25.7, 12: 30.4).
template <typename T, int D, int NC>
__global__ void __launch_bounds__(256, 3) kv4_score_kernel(SagaKv4Args a, uint32_t* __restrict__ keys, int per_warp) {
  constexpr int N = D / 32, NV = 4 * NC;
  __shared__ __align__(16) float qs[NV][32][N];  // a lane's channels are one load
  pdl_wait();
  const int G = a.Hq / a.pool.Hk;
  const int row = blockIdx.y;
  const int b = row / a.pool.Hk, kh = row % a.pool.Hk;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int pl = a.pool.page_len;
  const int len = min(max(a.lens[b], 0), a.max_pages * pl);
  const int pages = (len + pl - 1) / pl;
  // the kept pages at either end need no score
  const int c0 = a.keep_first + (int)blockIdx.x * 8 * per_warp, j1 = pages - a.keep_last;
  if (pages <= a.top || c0 >= j1) return;  // all are kept, or the row ends before this CTA
  const int j0 = c0 + warp * per_warp;
  const int n = min(per_warp, j1 - j0);
  int mine = 0;  // lane i has the warp's i-th page
  if (lane < n) {
    mine = a.page_table[(int64_t)b * a.pt_sb + j0 + lane];
    if (mine < 0 || mine >= a.pool.num_pages) {
      set_status(a.status, SAGA_STATUS_PAGE_RANGE);
      mine = 0;
    }
  }
  const T* q = reinterpret_cast<const T*>(a.q) + (int64_t)b * a.q_sb + (int64_t)kh * G * a.q_sh;
  auto stage = [&](int g0) {
    // one coalesced load of the queries per CTA: a warp's own 2-byte loads of all heads took longer than its pages
    __syncthreads();
    for (int x = threadIdx.x; x < NV * D; x += 256) {
      const int g = x / D, d = x % D;
      qs[g][d % 32][d / 32] = g0 + g < G ? Num<T>::to_f(q[(int64_t)(g0 + g) * a.q_sh + d]) : 0.f;
    }
    __syncthreads();
  };
  // the bounds of a batch of pages are on their way together, while the queries are staged or the batch
  // before it is scored
  __nv_bfloat16 lo[kScoreBatch][N], hi[kScoreBatch][N], lo_next[kScoreBatch][N], hi_next[kScoreBatch][N];
  auto fetch = [&](int p0) {
#pragma unroll
    for (int x = 0; x < kScoreBatch; ++x) {
      const int page = __shfl_sync(0xffffffffu, mine, (p0 + x) & 31);
      if (p0 + x < n) {
        const int64_t at = ((int64_t)page * a.pool.Hk + kh) * D + lane;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          lo_next[x][i] = reinterpret_cast<const __nv_bfloat16*>(a.pool.k_lo)[at + 32 * i];
          hi_next[x][i] = reinterpret_cast<const __nv_bfloat16*>(a.pool.k_hi)[at + 32 * i];
        }
      }
    }
  };
  fetch(0);
  for (int p0 = 0; p0 < per_warp; p0 += kScoreBatch) {  // the same trips for all warps: the staging has barriers
    if (p0 == 0) stage(0);
#pragma unroll
    for (int x = 0; x < kScoreBatch; ++x)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        lo[x][i] = lo_next[x][i];
        hi[x][i] = hi_next[x][i];
      }
    fetch(p0 + kScoreBatch);
    float best[kScoreBatch];
    bool nan[kScoreBatch];
#pragma unroll
    for (int x = 0; x < kScoreBatch; ++x) {
      best[x] = -INFINITY;
      nan[x] = false;
    }
    for (int g0 = 0; g0 < G; g0 += NV) {
      if (G > NV) stage(g0);
      // four heads at a time from shared memory, for all pages of the batch: with all heads in registers
      // one CTA filled an SM, and its warps waited for one another's loads
#pragma unroll 1
      for (int c = 0; c < NC; ++c) {
        f32x2 qv[4][N / 2];
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
          for (int i = 0; i < N / 2; ++i)
            qv[g][i] = reinterpret_cast<const f32x2*>(qs[4 * c + g][lane])[i];
        const bool real = g0 + 4 * c + lane / 8 < G;
#pragma unroll
        for (int x = 0; x < kScoreBatch; ++x) {
          if (p0 + x >= n) break;
          float s[4];
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            // lo <= hi, so the greater of the two products is the one that the sign of q picks
            f32x2 y[N / 2];
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
              float h0, h1, l0, l1;
              unpack2(mul2(qv[g][i], pack2(__bfloat162float(hi[x][2 * i]), __bfloat162float(hi[x][2 * i + 1]))), h0, h1);
              unpack2(mul2(qv[g][i], pack2(__bfloat162float(lo[x][2 * i]), __bfloat162float(lo[x][2 * i + 1]))), l0, l1);
              y[i] = pack2(fmaxf(h0, l0), fmaxf(h1, l1));
            }
            if constexpr (N == 4) y[0] = add2(y[0], y[N / 2 - 1]);  // channels d and d + 64
            float y0, y1;
            unpack2(y[0], y0, y1);
            s[g] = __fadd_rn(y0, y1);  // d and d + 32
          }
          const float t = warp_sums4(s);
          nan[x] |= real && t != t;
          if (real) best[x] = fmaxf(best[x], t);
        }
      }
    }
#pragma unroll
    for (int x = 0; x < kScoreBatch; ++x) {
      if (p0 + x >= n) break;
      uint32_t key = __reduce_max_sync(0xffffffffu, score_key(best[x]));
      if (__any_sync(0xffffffffu, nan[x])) key = kNanKey;
      if (lane == 0) keys[(int64_t)row * a.max_pages + j0 + p0 + x] = key;
    }
  }
}

// One CTA per (request, key head): the key of the last page to take by passes
// over 8 bits of the keys, then the pages above it and the lowest pages at it, in
// ascending order. The bits are those of the keys' own range (scores of one row
// share their upper bits: counting those would put all keys into one bin, one
// after the other), and the passes end once a bin is taken whole, for a thousand
// pages usually after two. 64 rows of up to 1025 pages take 7.6 us, latency alone:
// every pass is a round of counting and a scan by one warp between two barriers.
__global__ void __launch_bounds__(kTopThreads) kv4_top_kernel(SagaKv4Args a,
                                                              const uint32_t* __restrict__ row_keys) {
  constexpr int kTopWarps = kTopThreads / 32;
  __shared__ int hist[256];
  __shared__ int sh_bin, sh_left, sh_count;
  __shared__ uint32_t wred[2][kTopWarps];
  __shared__ int wsum[2][2][kTopWarps];
  __shared__ uint32_t keys[kTopKeys];
  pdl_wait();
  const int row = blockIdx.x;
  const int b = row / a.pool.Hk;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int pl = a.pool.page_len;
  const int given = a.lens[b];
  if (given > a.max_pages * pl && threadIdx.x == 0) set_status(a.status, SAGA_STATUS_PAGE_RANGE);
  const int len = min(max(given, 0), a.max_pages * pl);
  const int pages = (len + pl - 1) / pl;
  int32_t* out = a.blocks + (int64_t)row * a.top;
  if (threadIdx.x == 0) a.counts[row] = min(pages, a.top);
  if (pages <= a.top) {
    for (int i = threadIdx.x; i < a.top; i += kTopThreads) out[i] = i < pages ? i : -1;
    return;
  }
  const uint32_t* s = row_keys + (int64_t)row * a.max_pages;
  const int j0 = a.keep_first, j1 = pages - a.keep_last;  // the scored pages: [j0, j1)
  uint32_t least = 0xffffffffu, most = 0u;
  for (int j = j0 + threadIdx.x; j < j1; j += kTopThreads) {
    const uint32_t k = s[j];
    if (j < kTopKeys) keys[j] = k;
    least = min(least, k);
    most = max(most, k);
  }
  auto key_of = [&](int j) -> uint32_t { return j < kTopKeys ? keys[j] : s[j]; };
  least = __reduce_min_sync(0xffffffffu, least);
  most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 0) {
    wred[0][warp] = least;
    wred[1][warp] = most;
  }
  for (int i = threadIdx.x; i < 256; i += kTopThreads) hist[i] = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kTopWarps; ++w) {
    least = min(least, wred[0][w]);
    most = max(most, wred[1][w]);
  }
  int left = a.top - (a.keep_first + a.keep_last);  // scored pages to take among those that match `pre`
  int shift = j0 < j1 && most > least ? 32 - __clz(most - least) : 0;
  uint32_t pre = 0;  // key - least, shifted, of the bin that holds the last one
  while (shift > 0 && left > 0) {
    const int width = min(8, shift), up = shift;
    shift -= width;
    for (int j = j0 + threadIdx.x; j < j1; j += kTopThreads) {
      const uint32_t d = key_of(j) - least;
      if ((uint32_t)((uint64_t)d >> up) == pre) atomicAdd(&hist[(d >> shift) & ((1u << width) - 1u)], 1);
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
          sh_count = c[i];
        }
        above += c[i];
        hist[255 - 8 * lane - i] = 0;  // for the next pass
      }
    }
    __syncthreads();
    pre = (pre << width) | (uint32_t)sh_bin;
    left = sh_left;
    if (sh_count == left) break;  // the bin is taken whole
  }
  int done_gt = 0, done_eq = 0;  // pages above the key and at it so far
  int turn = 0;
  for (int base = 0; base < pages; base += kTopThreads, turn ^= 1) {
    const int j = base + threadIdx.x;
    const bool scored = j >= j0 && j < j1;
    const uint32_t d = scored ? (uint32_t)((uint64_t)(key_of(j) - least) >> shift) : 0u;  // shift: up to 32
    const bool gt = j < pages && (!scored || d > pre), eq = scored && d == pre;
    const unsigned bg = __ballot_sync(0xffffffffu, gt), be = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) {
      wsum[turn][0][warp] = __popc(bg);
      wsum[turn][1][warp] = __popc(be);
    }
    __syncthreads();  // the other half of wsum is written next: one barrier per round
    int g = done_gt, e = done_eq;
#pragma unroll
    for (int w = 0; w < kTopWarps; ++w) {
      if (w < warp) {
        g += wsum[turn][0][w];
        e += wsum[turn][1][w];
      }
      done_gt += wsum[turn][0][w];
      done_eq += wsum[turn][1][w];
    }
    const unsigned below = (1u << lane) - 1u;
    g += __popc(bg & below);
    e += __popc(be & below);
    if (gt || (eq && e < left)) out[g + min(e, left)] = j;
  }
}

}  // namespace

size_t kv4_select_workspace(const SagaKv4Args& a) {
  return ((size_t)a.B * a.pool.Hk * a.max_pages * sizeof(float) + 255) / 256 * 256 + 256;
}

int launch_kv4_select(const SagaKv4Args& a, cudaStream_t st) {
  uint32_t* keys = reinterpret_cast<uint32_t*>(a.workspace);
  const int rows = a.B * a.pool.Hk;
  const int G = a.Hq / a.pool.Hk;
  if (rows > 65535) return abi_fail(SAGA_ERR_UNSUPPORTED, "more than 65535 (request, key head) rows");
  if (a.max_pages > a.top) {
    // one page per warp where the SMs hold that many warps, else up to eight
    const int64_t warps = (int64_t)rows * a.max_pages;
    const int64_t held = 16ll * sm_count();
    const int per_warp = (int)std::min<int64_t>(kScorePages, (warps + held - 1) / held);
    const dim3 grid((a.max_pages + 8 * per_warp - 1) / (8 * per_warp), rows);
    auto go = [&](auto* t, auto d) {
      using T = std::remove_pointer_t<decltype(t)>;
      return kv4_launch("kv4_score_kernel",
                        G <= 4    ? kv4_score_kernel<T, d.value, 1>
                        : G <= 8  ? kv4_score_kernel<T, d.value, 2>
                        : G <= 12 ? kv4_score_kernel<T, d.value, 3>
                                  : kv4_score_kernel<T, d.value, 4>,
                        grid, 256, 0, st, a, keys, per_warp);
    };
    auto by_d = [&](auto* t) {
      return a.pool.D == 128 ? go(t, std::integral_constant<int, 128>()) : go(t, std::integral_constant<int, 64>());
    };
    const int rc = a.dtype == SAGA_BF16   ? by_d((__nv_bfloat16*)nullptr)
                   : a.dtype == SAGA_FP16 ? by_d((__half*)nullptr)
                                          : by_d((float*)nullptr);
    if (rc) return rc;
  }
  return kv4_launch("kv4_top_kernel", kv4_top_kernel, dim3(rows), kTopThreads, 0, st, a, keys);
}

}  // namespace saga
