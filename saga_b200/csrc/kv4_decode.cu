// Attention of one query position per request over the 4-bit paged cache.
//
// With x = s_g * code + z_g per group g of 64 channels,
//   q.k   = sum_g s_g (q_g . code_g) + z_g sum(q_g)
//   out_d = (sum_t p_t s_{t,g(d)} code_{t,d} + sum_t p_t z_{t,g(d)}) / sum_t p_t,
// so the matrix products run on the bare codes and the scales touch only one
// value per (position, query head) and group.
//
// Work: an item is a (request, key head, up to 16 of its query heads). Its
// positions are tiles of 32; the tiles of all items form one list, of which
// every CTA takes an equal run (lengths are read on the device), where an item
// counts for some tiles more than it has, since a CTA pays for each. A warp works
// alone: it copies its next tiles into a ring of its own with one bulk copy per
// head, and holds a running maximum, sums and outputs in registers. The warps
// of a CTA meet at the end of an item; items cut by CTA borders leave partial
// results that kv4_combine_kernel joins.
//
// Products: mma.sync m16n8k16 in fp16 with operands built in registers. A code
// masked out of its word, unshifted, is a subnormal fp16: bits 0-3 are code *
// 2^-24, bits 4-7 are code * 2^-20, so eight codes become four operand
// registers with one shift and four ANDs (for fp32 tensors they are made normal
// numbers first, see whole()). Feeding tcgen05 instead would put the
// widened codes through shared memory (4x the bytes of the cache, written and
// read), which at the HBM rate would already fill its bandwidth.
//   scores: A = queries (slots x channels), B = codes (channels x positions)
//   output: A = codes transposed (ldmatrix.trans: channels x positions),
//           B = weights (positions x slots): the scores' accumulators have
//           exactly this layout, so the weights never leave their lane.
//
// Measured, per call with the join: 64 x 65,600 positions, 12 query, 1 key and 4
// value heads of 128, bf16, 361 us for 1.51 GB, 4.2 TB/s (337 us back to back on
// one cache); 8 x 32,768, 12/1/2 heads, 29.4 us for 56.6 MB, 1.9 TB/s (27.7 us
// back to back, from L2). What bounds it is not the memory but the work per code:
// the schedulers issue in 43 % of the cycles and the logical operations take 34 %
// of theirs, and with 254 registers a thread there are two warps per scheduler to
// cover the products' latency. Twelve warps spill and gain nothing; scores in
// e4m3, whose instruction is twice as fast, need a further term per query and
// its registers (31 us instead of 27, back to back).
#include <algorithm>

#include "kv4.cuh"
#include "tc.cuh"

namespace saga {

namespace {

constexpr int kDecWarps = 8;
constexpr int kDecThreads = kDecWarps * 32;
constexpr int kMaxSlots = 16;       // query heads of an item
constexpr int kMaxRing = 4;         // stages of a warp's ring
constexpr int kMinTiles = 4;        // tiles of a CTA's run, at least: one warp per scheduler
// Tiles that an item's own cost counts for when the work is dealt out: the start of its copies and the meeting
// of the warps take about 5 us, a round of eight tiles 2 to 3 us. Sixteen ragged rows of up to 16,512 positions
// take 19.0 us with 0, 15.8 with 8, 15.6 with 16 and 15.5 with 32; 64 ragged rows of up to 2048 positions 24.8,
// 18.2, 18.5 and 21.1.
constexpr int kItemTiles = 16;
constexpr int kRingBytes = 216 * 1024;  // of all warps; static shared memory has the rest
constexpr float kHead = 12.f;     // log2 of the greatest weight where the stabilisers were last set
constexpr float kSlack = 15.f;    // log2 of the greatest weight, and of the greatest p, that is left as it is
constexpr float kLow = 2048.f;    // SPLIT: the second term of a weight is held this much greater
// -16 * 15, and -15 with it, in units of 2^-24, twice
constexpr uint32_t kMinus240 = 0x80f080f0u, kMinus255 = 0x80ff80ffu;
constexpr float kNegInf = -INFINITY;

// Query heads of a key head are cut into slot groups: consecutive heads, at most
// `slots` of them and at most `vheads` value heads (the size of a ring stage).
struct SlotGroup {
  int h0, n;  // first query head, number of heads
};
__host__ __device__ inline SlotGroup slot_group(int kh, int sg, int G, int Gv, int slots, int vheads) {
  int h = kh * G;
  const int end = h + G;
  for (;; --sg) {
    const int stop = ((h / Gv) + vheads) * Gv;  // first head of the value head past the limit
    int n = end - h;
    if (n > slots) n = slots;
    if (n > stop - h) n = stop - h;
    if (sg == 0 || h + n >= end) return {sg == 0 ? h : end, sg == 0 ? n : 0};
    h += n;
  }
}

struct DecodePlan4 {
  SagaKv4Args a;
  int groups;      // slot groups per key head
  int vheads;      // value heads of a slot group, at most
  int stages;      // ring stages per warp
  int ring_bytes;  // of one warp
  int tpp_shift;   // log2 of the tiles per page
  float* part_o;   // [grid][2][slots][D] numerators of cut items
  float* part_ml;  // [grid][2][slots][2] their maxima and sums
  long long* prefix;  // [rows + 1] weight of the items before a (request, key head) row
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  // volatile: it must not be moved in front of the (warp-uniform) branches around it
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
      "%2, %3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// The same with nothing added: the accumulators need not be cleared first.
__device__ __forceinline__ void mma16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, "
      "%10, %10};\n"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// log2 of a positive bfloat16 scale, up to 0.09 below it (its bits are a
// piecewise linear logarithm). It only places the stabilisers.
__device__ __forceinline__ float rough_log2(uint32_t bf16_bits) {
  return fmaf(__uint_as_float(0x4b000000u | bf16_bits), 0x1p-7f, -65663.f);
}
// The greatest of each over the four lanes of a quad.
template <int N>
__device__ __forceinline__ void quad_max(float (&x)[N]) {
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {
    float y[N];
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = __shfl_xor_sync(0xffffffffu, x[i], o);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = fmaxf(x[i], y[i]);
  }
}
// 2^x of a whole number from -126 to 126: it is put where the exponent lies.
__device__ __forceinline__ float exp2_whole(float x) {
  return __uint_as_float(__float_as_uint(x + (12582912.f + 127.f)) << 23);
}
// 2 code - 15 of a byte's codes (the upper one's times 16), in units of 2^-24: exact in fp16.
__device__ __forceinline__ uint32_t centre(uint32_t codes, uint32_t minus) {
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&codes), __floats2half2_rn(2.f, 2.f),
                            *reinterpret_cast<const __half2*>(&minus));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// SPLIT: codes as normal fp16 numbers (those of bits 0-3, or 16 times those of bits 4-7), and 32 code - 240 of bits
// 4-7; set into the low bits of 1024 they are exact. The tensor cores align the products of a sum by the exponents
// of their operands, a subnormal's being that of 2^-14: up to ten bits of a product with a code of 2^-24 are lost
// beside the greatest query or weight. Terms of 22 bits feel that (fp32 errors 3 to 4e-6 with subnormals, 3 to 5e-7
// without; 4 x 4099 positions 13.0 and 13.4 us), one term of 11 bits does not (fp16 errors are the same both ways, and
// 8 x 32,768 positions take 29.3 and 29.8 us).
__device__ __forceinline__ uint32_t whole(uint32_t codes) {
  const uint32_t u = codes | 0x64006400u;
  const __half2 r = __hadd2(*reinterpret_cast<const __half2*>(&u), __floats2half2_rn(-1024.f, -1024.f));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t centre16(uint32_t codes) {
  const uint32_t u = codes | 0x64006400u;
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&u), __floats2half2_rn(2.f, 2.f),
                            __floats2half2_rn(-2288.f, -2288.f));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// The scale words of positions pos and pos + 1 (pos even).
template <int NG>
__device__ __forceinline__ void load_meta(const uint8_t* meta, int pos, uint32_t (&w)[2][NG]) {
  if constexpr (NG == 2) {
    const uint4 t = *reinterpret_cast<const uint4*>(meta + pos * 8);
    w[0][0] = t.x;
    w[0][1] = t.y;
    w[1][0] = t.z;
    w[1][1] = t.w;
  } else {
    const uint2 t = *reinterpret_cast<const uint2*>(meta + pos * 4);
    w[0][0] = t.x;
    w[1][0] = t.y;
  }
}
__device__ __forceinline__ void store_out(void* o, int dt, int64_t i, float x) {
  if (dt == SAGA_BF16) reinterpret_cast<__nv_bfloat16*>(o)[i] = __float2bfloat16_rn(x);
  else if (dt == SAGA_FP16) reinterpret_cast<__half*>(o)[i] = __float2half_rn(x);
  else reinterpret_cast<float*>(o)[i] = x;
}

// Positions of a row and its number of tiles (of every slot group).
struct RowInfo {
  int start, len, tiles, first;  // first: dense, the tile that holds `start`
};
__device__ __forceinline__ RowInfo row_info(const SagaKv4Args& a, int r) {
  const int b = r / a.pool.Hk;
  RowInfo i;
  i.len = min(max(a.lens[b], 0), a.max_pages * a.pool.page_len);
  i.start = a.starts ? max(a.starts[b], 0) : 0;
  i.first = i.start / kKv4Tile;
  if (i.start >= i.len) i.tiles = 0;
  else if (a.blocks) i.tiles = min(max(a.counts[r], 0), a.top) * (a.pool.page_len / kKv4Tile);
  else i.tiles = (i.len + kKv4Tile - 1) / kKv4Tile - i.first;
  return i;
}

// What an item of the row counts for when the work is dealt out: kItemTiles, then its tiles.
__device__ __forceinline__ int item_weight(const RowInfo& i) { return i.tiles ? kItemTiles + i.tiles : 0; }

// Quotient of numbers that are not negative; 32 bits where they fit, since a 64-bit division takes about a
// hundred instructions.
__device__ __forceinline__ long long divide(long long a, long long b) {
  return (a | b) >> 32 ? a / b : (long long)((uint32_t)a / (uint32_t)b);
}
__device__ __forceinline__ long long tiles_per_cta(long long total, int grid) {
  return max(divide(total + grid - 1, grid), (long long)kMinTiles);
}

// D: head_dim; NT: tiles of eight slots; SPLIT: queries and weights as two fp16
// terms each (fp32 tensors, 22 significant bits). bf16 and fp16 tensors take
// weights of one fp16 term, which is a choice: its rounding is averaged over the
// positions, and a second term would double the output's products. Relative rms
// errors (and those of binary32 arithmetic rounded once): fp16 2.7e-4 (2.1e-4),
// bf16 1.67e-3 (1.65e-3), fp32 3 to 5e-7 (5 to 15e-7).
template <int D, int NT, bool SPLIT>
__global__ void __launch_bounds__(kDecThreads, 1) kv4_decode_kernel(const DecodePlan4 p) {
  constexpr int NG = D / 64, CH = D / 32, NP = SPLIT ? 2 : 1, SLOTS = 8 * NT;
  constexpr int TB = kv4_tile_bytes(D);
  constexpr int META = kKv4Tile * (D / 2);
  // Whether channel rows 0-7 of a product take both codes of a byte, c + 16 c' (rows 8-15 have 16 c' and are
  // taken off at the end): an AND less per code, four bits less of the sums.
  constexpr bool kPairs = !SPLIT;
  // SPLIT: the stabilisers are whole numbers, so that the factors between them are exact. With one term the
  // greatest weight is put just below a power of two instead, where it is rounded least (rough_log2 is up to 0.09
  // below): fp16 errors 2.7e-4 instead of 3.0e-4.
  constexpr bool kWhole = SPLIT;
  // what a product's one is, in channel rows 0-7 and 8-15
  constexpr float kUnitE = SPLIT ? 0x1p-5f : 0x1p23f, kUnitH = SPLIT ? 0x1p-5f : 0x1p19f;
  constexpr int RP = D + 4;   // pitch of a warp's outputs when the warps meet
  constexpr int QP = D + 8;   // pitch of the queries
  constexpr int QT = 16, QC = D / QT;  // threads per slot's query, channels of each
  extern __shared__ __align__(128) uint8_t ring_all[];
  __shared__ __align__(16) __half qs[NP][kMaxSlots][QP];
  __shared__ uint64_t full[kDecWarps][kMaxRing];
  __shared__ long long scan_sm[kDecWarps];
  __shared__ long long sh_row_base;
  __shared__ int sh_row;
  __shared__ int slot_head[kMaxSlots], slot_vh[kMaxSlots];
  __shared__ uint32_t sh_on;
  __shared__ float q_unit[kMaxSlots], q_sum[kMaxSlots][2];
  __shared__ float sm_m[kDecWarps][kMaxSlots], sm_l[kDecWarps][kMaxSlots], sm_f[kDecWarps][kMaxSlots];

  const SagaKv4Args& a = p.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r8 = lane >> 2, c4 = lane & 3;
  const int Hk = a.pool.Hk, G = a.Hq / Hk, Gv = a.Hq / a.pool.Hv;
  const int rows = a.B * Hk;
  const int tpp_shift = p.tpp_shift, tpp_mask = (1 << tpp_shift) - 1;

  if (lane == 0) {
    for (int s = 0; s < kMaxRing; ++s) mbar_init(&full[warp][s], 1);
    mbar_fence_init();
  }

  pdl_wait();
  // ---- this CTA's run of tiles: [run, run_end), and the row it begins in
  long long total = 0;
  if (rows > kDecThreads) {
    for (int r = threadIdx.x; r < rows; r += kDecThreads) total += item_weight(row_info(a, r));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (lane == 0) scan_sm[warp] = total;
    __syncthreads();
    total = 0;
    for (int w = 0; w < kDecWarps; ++w) total += scan_sm[w];
    total *= p.groups;
    __syncthreads();
  }
  long long run = 0, run_end = 0, base = 0;
  const bool writes_prefix = blockIdx.x == 0;
  for (int r0 = 0; r0 < rows; r0 += kDecThreads) {
    const int r = r0 + threadIdx.x;
    const long long t = r < rows ? (long long)item_weight(row_info(a, r)) * p.groups : 0;
    long long inc = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) scan_sm[warp] = inc;
    __syncthreads();
    long long before = base;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
      if (w < warp) before += scan_sm[w];
      base += scan_sm[w];
    }
    before += inc - t;
    if (r0 == 0) {
      if (rows <= kDecThreads) total = base;
      const long long per = tiles_per_cta(total, gridDim.x);
      run = per * blockIdx.x;
      run_end = min(run + per, total);
    }
    if (r < rows && run >= before && run < before + t) {
      sh_row = r;
      sh_row_base = before;
    }
    if (writes_prefix && r < rows) {
      p.prefix[r] = before;
      if (r == rows - 1) p.prefix[rows] = before + t;
    }
    __syncthreads();
    if (!writes_prefix && (run >= run_end || base > run)) break;
  }
  if (run >= run_end) return;
  int row = sh_row;
  long long row_base = sh_row_base;

  uint8_t* ring = ring_all + (size_t)warp * p.ring_bytes;
  const uint32_t ring_s = smem_addr(ring);
  const int stage_bytes = (1 + p.vheads) * TB;
  // ring positions and parities of the next tile to issue and to consume
  int st_i = 0, st_c = 0;
  uint32_t par_c = 0;
  bool alive = true;
  int have_kh = -1, have_sg = -1;

  while (run < run_end) {
    // ---- the item: row, slot group, tiles [t0, t1) of the row
    RowInfo ri = row_info(a, row);
    while (run >= row_base + (long long)item_weight(ri) * p.groups) {
      row_base += (long long)item_weight(ri) * p.groups;
      ri = row_info(a, ++row);
    }
    int sg = 0;
    long long tile_base = row_base + kItemTiles;  // of the item's tile 0
    while (run >= tile_base + ri.tiles) {
      tile_base += item_weight(ri);
      ++sg;
    }
    const int t0 = (int)max(run - tile_base, 0ll);
    const int t1 = (int)min((long long)ri.tiles, run_end - tile_base);
    if (t1 <= t0) break;  // the run ends before the item's first tile
    const int b = row / Hk, kh = row - b * Hk;
    const SlotGroup grp = slot_group(kh, sg, G, Gv, SLOTS, p.vheads);
    const int vh0 = grp.h0 / Gv;
    const int nvh = grp.n ? (grp.h0 + grp.n - 1) / Gv - vh0 + 1 : 0;

    // ---- the warp's tiles: t0 + warp, + kDecWarps, ...
    const int mine = alive ? max(t1 - t0 - warp + kDecWarps - 1, 0) / kDecWarps : 0;
    const int32_t* blocks = a.blocks ? a.blocks + (int64_t)row * a.top : nullptr;
    // tile in the pool and first position of the warp's tile k (lane k % 32 of a batch of 32)
    auto locate = [&](int k, int& ptile, int& pos) {
      ptile = 0;
      pos = 0x7fffff00;  // masked altogether
      if (k >= mine) return;
      int t = t0 + warp + k * kDecWarps;
      if (!blocks) t += ri.first;
      int pi = t >> tpp_shift;
      const int off = t & tpp_mask;
      if (blocks) pi = blocks[pi];
      if (pi < 0 || pi >= a.max_pages) return;
      int page = a.page_table[(int64_t)b * a.pt_sb + pi];
      if (page < 0 || page >= a.pool.num_pages) {
        set_status(a.status, SAGA_STATUS_PAGE_RANGE);
        page = 0;
      }
      ptile = (page << tpp_shift) + off;  // the host checks that the pool's tiles fit an int
      pos = ((pi << tpp_shift) + off) * kKv4Tile;
    };
    int pg0, ps0, pg1, ps1;
    locate(lane, pg0, ps0);
    locate(32 + lane, pg1, ps1);
    // lane 0 copies the tile's keys, lane 1 + j those of value head j
    const bool copies = lane <= nvh;
    const uint8_t* src0 = reinterpret_cast<const uint8_t*>(lane == 0 ? a.pool.k : a.pool.v);
    const int src_heads = lane == 0 ? Hk : a.pool.Hv, src_head = lane == 0 ? kh : vh0 + lane - 1;
    auto issue = [&](int k) {  // k: the warp's tile, in order
      if ((k & 31) == 0 && k > 0) {
        pg0 = pg1;
        ps0 = ps1;
        locate(k + 32 + lane, pg1, ps1);
      }
      const int ptile = __shfl_sync(0xffffffffu, pg0, k & 31);
      uint64_t* bar = &full[warp][st_i];
      if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)((1 + nvh) * TB));
      __syncwarp();
      if (copies) {
        const int64_t page = ptile >> tpp_shift;
        const int64_t at = ((page * src_heads + src_head) << tpp_shift) + (ptile & tpp_mask);
        bulk_load(ring + st_i * stage_bytes + lane * TB, src0 + at * TB, TB, bar);
      }
      if (++st_i == p.stages) st_i = 0;
    };
    // positions of the tiles being consumed: the batch that `issue` holds may be one ahead
    int cp0 = ps0, cp1 = ps1;

    // ---- slots of the item's query heads
    if (kh != have_kh || sg != have_sg) {
      if (warp == 0) {
        // a value head's slots stay inside one tile of eight where that fits, since
        // its codes are multiplied with every tile that has one of its slots
        int head = -1, vh = -1;
        for (int pass = 0; pass < 2; ++pass) {
          int at = 0, h = grp.h0;
          head = vh = -1;
          for (int v = 0; h < grp.h0 + grp.n; ++v) {
            const int n = min((vh0 + v + 1) * Gv, grp.h0 + grp.n) - h;
            if (pass == 0 && (at & 7) && (at & 7) + min(n, 8) > 8) at = (at + 7) & ~7;
            if (at + n > SLOTS) break;
            if (lane >= at && lane < at + n) {
              head = h + lane - at;
              vh = v;
            }
            at += n;
            h += n;
          }
          if (h >= grp.h0 + grp.n) break;
        }
        if (lane < kMaxSlots) {
          slot_head[lane] = head;
          slot_vh[lane] = vh;
        }
        // bits 2j, 2j + 1: slot tiles that hold slots of value head j
        const uint32_t on = __reduce_or_sync(0xffffffffu, vh < 0 ? 0u : 1u << (2 * vh + lane / 8));
        if (lane == 0) sh_on = on;
      }
      have_kh = kh;
      have_sg = sg;
      __syncthreads();
    }

    // ---- queries, scaled by a power of two that brings the greatest |q| of a head into [2^14, 2^15).
    // Order within eight channels: (0, 4) (1, 5) (2, 6) (3, 7), the pairs in which codes leave a word;
    // odd channels' codes are read 16 times too great.
    {
      const int s = min((int)threadIdx.x / QT, kMaxSlots - 1), i0 = (threadIdx.x % QT) * QC;
      const int h = s < SLOTS ? slot_head[s] : -1;
      const int64_t at = (int64_t)b * a.q_sb + (int64_t)h * a.q_sh + i0;
      float v[QC], amax = 0.f;
#pragma unroll
      for (int i = 0; i < QC; ++i) v[i] = 0.f;
      if (h >= 0) {
        if (a.dtype == SAGA_BF16) {
#pragma unroll
          for (int i = 0; i < QC; ++i) v[i] = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.q)[at + i]);
        } else if (a.dtype == SAGA_FP16) {
#pragma unroll
          for (int i = 0; i < QC; ++i) v[i] = __half2float(reinterpret_cast<const __half*>(a.q)[at + i]);
        } else {
#pragma unroll
          for (int i = 0; i < QC; ++i) v[i] = reinterpret_cast<const float*>(a.q)[at + i];
        }
      }
      // the first copies leave while the queries arrive
      const int ahead = min(p.stages - 1, mine);
      for (int k = 0; k < ahead; ++k) issue(k);
#pragma unroll
      for (int i = 0; i < QC; ++i) amax = fmaxf(amax, fabsf(v[i]));
#pragma unroll
      for (int o = QT / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      // e = 14 - floor(log2 amax), kept where 2^e and 2^-e are normal; an infinite or NaN query stays itself
      const int ex = (int)(__float_as_uint(amax) >> 23);
      const int e = ex == 0 ? 126 : ex == 255 ? 0 : min(141 - ex, 126);
      const float up = __uint_as_float((uint32_t)(127 + e) << 23), down = __uint_as_float((uint32_t)(127 - e) << 23);
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < QC; ++i) {
        const int d = i0 + i, n = d & 7;
        const float x = v[i] * up;
        const float hi = __half2float(__float2half_rn(x));
        const float f = n & 1 ? 0.0625f : 1.f;
        const int to = (d & ~7) + 2 * (n & 3) + (n >> 2);
        qs[0][s][to] = __float2half_rn(hi * f);
        sum += hi;
        if constexpr (SPLIT) {
          const float lo = __half2float(__float2half_rn(x - hi));
          qs[1][s][to] = __float2half_rn(lo * f);
          sum += lo;
        }
      }
      // the threads of a group of 64 channels
#pragma unroll
      for (int o = 64 / QC / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (i0 % 64 == 0) q_sum[s][i0 / 64] = sum;
      if (i0 == 0) q_unit[s] = a.scaling * 1.4426950408889634f * down;  // scores in powers of two
    }
    __syncthreads();
    f32x2 fh[NT], Qz[NT][NG];    // each value twice
    int vhl[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int s = r8 + 8 * i;
      vhl[i] = slot_vh[s];
      const float unit = q_unit[s];
      fh[i] = pack2(unit * (SPLIT ? 1.f : 0x1p24f), unit * (SPLIT ? 1.f : 0x1p24f));
#pragma unroll
      for (int g = 0; g < NG; ++g) Qz[i][g] = pack2(q_sum[s][g] * unit, q_sum[s][g] * unit);
    }
    const uint32_t on_all = sh_on;

    f32x2 o[NT][D / 16][2];  // channel rows r8 and r8 + 8, two slots each
    float mrun[NT], shift[NT][NG];  // the stabilisers
    f32x2 lsum[NT], zsum[NT][NG];  // over the even and the odd positions
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int m = 0; m < D / 16; ++m) o[i][m][0] = o[i][m][1] = 0ull;
      mrun[i] = kNegInf;
      lsum[i] = 0ull;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        zsum[i][g] = 0ull;
        shift[i][g] = 0.f;
      }
    }

    for (int k = 0; k < mine; ++k) {
      if (k + p.stages - 1 < mine) issue(k + p.stages - 1);
      if ((k & 31) == 0 && k > 0) {
        cp0 = cp1;
        cp1 = ps1;  // `issue` has moved on to the batch after this one, if there is one
      }
      // the lanes vote: a copy that arrives near the limit must not leave some of them behind
      if (!__all_sync(0xffffffffu, mbar_wait(&full[warp][st_c], par_c, a.status))) {
        // the copies in flight get one more bounded wait each; then this warp only keeps the barriers
        for (int x = k; x < min(k + p.stages, mine); ++x) {
          mbar_wait(&full[warp][st_c], par_c, a.status);
          if (++st_c == p.stages) {
            st_c = 0;
            par_c ^= 1u;
          }
        }
        __syncwarp();
        alive = false;
        break;
      }
      const uint32_t ks = ring_s + st_c * stage_bytes;
      uint8_t* kt = ring + st_c * stage_bytes;
      if (++st_c == p.stages) {
        st_c = 0;
        par_c ^= 1u;
      }
      const int pos0 = __shfl_sync(0xffffffffu, cp0, k & 31);
      const bool edge = pos0 < ri.start || pos0 + kKv4Tile > ri.len;
      if (edge) {  // whatever a masked row holds must not meet its zero weight
        if (pos0 + lane < ri.start || pos0 + lane >= ri.len) {
          for (int u = 0; u <= nvh; ++u)
#pragma unroll
            for (int g = 0; g < NG; ++g) *reinterpret_cast<uint32_t*>(kt + u * TB + kv4_meta_off<D>(lane, g)) = 0u;
        }
        fence_proxy_async_smem();  // before the stage's next copy
        __syncwarp();
      }

      // ---- scores of 32 positions: l[i][j] = slot r8 + 8i, positions 8j + 2 c4 and the next
      f32x2 l[NT][4];
      {
        uint32_t kreg[4][CH];
        if constexpr (D == 128) {
#pragma unroll
          for (int j = 0; j < 4; ++j) ldsm4(kreg[j], ks + kv4_chunk_off<D>(8 * j + (lane & 7), lane >> 3));
        } else {
#pragma unroll
          for (int j = 0; j < 4; j += 2) {
            uint32_t t[4];
            ldsm4(t, ks + kv4_chunk_off<D>(8 * (j + (lane >> 4)) + (lane & 7), (lane >> 3) & 1));
            kreg[j][0] = t[0];
            kreg[j][1] = t[1];
            kreg[j + 1][0] = t[2];
            kreg[j + 1][1] = t[3];
          }
        }
        // the chunks of a group share accumulators; in fp32 (SPLIT) every chunk is rounded by itself
        constexpr int STEP = SPLIT ? 1 : 2;
#pragma unroll
        for (int c0 = 0; c0 < CH; c0 += STEP) {
          const int g = c0 / 2;
          // consecutive products go to different accumulators: one chain waits for itself at every step
          float acc[4][4];
#pragma unroll
          for (int ch = c0; ch < c0 + STEP; ++ch)
#pragma unroll
            for (int t = 0; t < NP; ++t) {
              uint32_t q[NT][4];  // pairs of channels (0, 4) (1, 5) (2, 6) (3, 7) of slots r8 + 8i
#pragma unroll
              for (int i = 0; i < NT; ++i) {
                const uint4 x = *reinterpret_cast<const uint4*>(&qs[t][r8 + 8 * i][32 * ch + 8 * c4]);
                q[i][0] = x.x;
                q[i][1] = x.y;
                q[i][2] = x.z;
                q[i][3] = x.w;
              }
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const uint32_t w = h ? kreg[j][ch] >> 8 : kreg[j][ch];
                  const uint32_t x0 = SPLIT ? whole(w & 0x000f000fu) : w & 0x000f000fu;
                  const uint32_t x1 = SPLIT ? whole(w & 0x00f000f0u) : w & 0x00f000f0u;
                  const uint32_t a1 = NT == 2 ? q[NT - 1][2 * h] : 0u, a3 = NT == 2 ? q[NT - 1][2 * h + 1] : 0u;
                  if (ch == c0 && t == 0 && h == 0) mma16_first(acc[j], q[0][2 * h], a1, q[0][2 * h + 1], a3, x0, x1);
                  else mma16(acc[j], q[0][2 * h], a1, q[0][2 * h + 1], a3, x0, x1);
                }
            }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t mw[2][NG];
            load_meta<NG>(kt + META, 8 * j + 2 * c4, mw);
            const f32x2 ms = pack2(kv4_scale(mw[0][g]), kv4_scale(mw[1][g]));
            const f32x2 mz = pack2(kv4_zero(mw[0][g]), kv4_zero(mw[1][g]));
#pragma unroll
            for (int i = 0; i < NT; ++i) {
              const f32x2 y = mul2(fh[i], ms);
              const f32x2 z = c0 == 0          ? mul2(mz, Qz[i][g])
                              : c0 % 2 == 0 ? fma2(mz, Qz[i][g], l[i][j])
                                            : l[i][j];
              l[i][j] = fma2(y, pack2(acc[j][2 * i], acc[j][2 * i + 1]), z);
            }
          }
        }
      }
      if (edge) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int pos = pos0 + 8 * j + 2 * c4;
          const bool m0 = pos < ri.start || pos >= ri.len, m1 = pos + 1 < ri.start || pos + 1 >= ri.len;
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            float y0, y1;
            unpack2(l[i][j], y0, y1);
            l[i][j] = pack2(m0 ? kNegInf : y0, m1 ? kNegInf : y1);
          }
        }
      }

      // ---- stabilisers. p = 2^(score - mrun) is of the scores alone; the weights p * s of group g are held
      // 2^shift[g] times greater, so that a group of small values is as exact beside one of great values as by
      // itself. Both are changed only when needed: p of at most 2^kSlack and weights of at most 2^kSlack are
      // left as they are. Whether they are is asked of a bound, the greatest score of a lane's positions with
      // the greatest of their scales.
      bool raise = false;
      float top_l[NT];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const uint8_t* vm = kt + (1 + max(vhl[i], 0)) * TB + META;
        uint32_t top[NG];
        float y = kNegInf;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t vw[2][NG];
          load_meta<NG>(vm, 8 * j + 2 * c4, vw);
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const uint32_t t = max_u16x2(vw[0][g], vw[1][g]);
            top[g] = j == 0 ? t : max_u16x2(top[g], t);
          }
          float y0, y1;
          unpack2(l[i][j], y0, y1);
          y = fmaxf(y, fmaxf(y0, y1));
        }
        top_l[i] = y;
        y -= mrun[i];
        raise |= y > kSlack;
#pragma unroll
        for (int g = 0; g < NG; ++g) raise |= y + shift[i][g] + rough_log2(top[g] & 0xffffu) > kSlack;
      }
      if (__any_sync(0xffffffffu, raise)) {
        // New ones put the greatest score at or below 0 and the greatest weight, now position by position, at
        // 2^kHead, so that weights far below it are still normal in fp16 (11 significant bits down to 2^-14).
        float down[NT], most[NT][NG];
        quad_max(top_l);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const float mn = fmaxf(mrun[i], kWhole ? ceilf(top_l[i]) : top_l[i]);
          down[i] = mn == kNegInf ? 0.f : mrun[i] - mn;
          mrun[i] = mn;
          const uint8_t* vm = kt + (1 + max(vhl[i], 0)) * TB + META;
#pragma unroll
          for (int g = 0; g < NG; ++g) most[i][g] = kNegInf;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t vw[2][NG];
            load_meta<NG>(vm, 8 * j + 2 * c4, vw);
            float y0, y1;
            unpack2(l[i][j], y0, y1);
#pragma unroll
            for (int g = 0; g < NG; ++g)
              most[i][g] = fmaxf(most[i][g], fmaxf(y0 - mn + rough_log2(vw[0][g] & 0xffffu),
                                                   y1 - mn + rough_log2(vw[1][g] & 0xffffu)));
          }
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) quad_max(most[i]);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const float f = ex2(down[i]);
          const f32x2 ff = pack2(f, f);
          lsum[i] = mul2(lsum[i], ff);
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            zsum[i][g] = mul2(zsum[i][g], ff);
            // a scale of 0 (a group that stands for NaN) leaves the shift within what 2^shift can be
            const float to =
                fmaxf(fminf(fminf(shift[i][g] - down[i], kHead - (kWhole ? ceilf(most[i][g]) : most[i][g] + 0.09f)),
                            126.f), -126.f);
            const float fg = ex2(down[i] + (to - shift[i][g]));
            shift[i][g] = to;
            const f32x2 fo = pack2(__shfl_sync(0xffffffffu, fg, 8 * c4), __shfl_sync(0xffffffffu, fg, 8 * c4 + 4));
#pragma unroll
            for (int m = 4 * g; m < 4 * g + 4; ++m) {
              o[i][m][0] = mul2(o[i][m][0], fo);
              o[i][m][1] = mul2(o[i][m][1], fo);
            }
          }
        }
      }

      // ---- weights p * s of 32 positions, as B operands of two steps of 16
      uint32_t wb[2][NP][NT][NG][2];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const float ms = mrun[i] == kNegInf ? 0.f : -mrun[i];
        const f32x2 ms2 = pack2(ms, ms), middle = pack2(7.5f, 7.5f);
        const uint8_t* vm = kt + (1 + max(vhl[i], 0)) * TB + META;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t vw[2][NG];
          load_meta<NG>(vm, 8 * j + 2 * c4, vw);
          float p0, p1;
          unpack2(add2(l[i][j], ms2), p0, p1);
          const f32x2 pp = pack2(ex2(p0), ex2(p1));
          lsum[i] = add2(lsum[i], pp);
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const f32x2 w = mul2(pp, pack2(kv4_scale(vw[0][g]), kv4_scale(vw[1][g])));
            // sum of p (z + 7.5 s): the products below take code - 7.5
            zsum[i][g] = fma2(pp, pack2(kv4_zero(vw[0][g]), kv4_zero(vw[1][g])), zsum[i][g]);
            zsum[i][g] = fma2(middle, w, zsum[i][g]);
            const float up = kWhole ? exp2_whole(shift[i][g]) : ex2(shift[i][g]);
            float w0, w1;
            unpack2(mul2(w, pack2(up, up)), w0, w1);
            uint32_t& hi = wb[j >> 1][0][i][g][j & 1];
            hi = pack_half2(w0, w1);
            if constexpr (SPLIT) {
              const __half2 hv = *reinterpret_cast<const __half2*>(&hi);
              wb[j >> 1][NP - 1][i][g][j & 1] =
                  pack_half2((w0 - __low2float(hv)) * kLow, (w1 - __high2float(hv)) * kLow);
            }
          }
        }
      }

      // ---- output. The tensor cores' sums are not rounded to nearest, so 32 positions are summed there
      // and the running sum is added outside; and the codes are taken about their middle (7.5), since
      // what they have in common grows with the positions, and with it the error, faster than the result.
      for (int v = 0; v < nvh; ++v) {
        const uint32_t vs = ks + (1 + v) * TB + kv4_chunk_off<D>(8 * ((lane >> 3) & 1) + (lane & 7), lane >> 4);
        const uint32_t on = on_all >> (2 * v);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          if ((on >> i & 1u) == 0u) continue;
          const uint32_t mine_v = vhl[i] == v ? 0xffffffffu : 0u;  // slots of other value heads get zero weights
          // rows 16 further have the same swizzle; group g's two chunks are those of group 0 with bit 5 flipped
          uint32_t t[NG][2][4];
#pragma unroll
          for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int jj = 0; jj < 2; ++jj) ldsm4t(t[g][jj], (vs ^ (g << 5)) + jj * 16 * (D / 2));
          uint32_t wv[NG][2][NP][2];
#pragma unroll
          for (int jj = 0; jj < 2; ++jj)
#pragma unroll
            for (int n = 0; n < NP; ++n)
#pragma unroll
              for (int g = 0; g < NG; ++g) {
                wv[g][jj][n][0] = wb[jj][n][i][g][0] & mine_v;
                wv[g][jj][n][1] = wb[jj][n][i][g][1] & mine_v;
              }
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            // products y = 2x + m: chunk 2g + x (positions 0-7 in t[2x], 8-15 in t[2x + 1]), bytes m and m + 2
            float s[NP][4][4];
#pragma unroll
            for (int jj = 0; jj < 2; ++jj)
#pragma unroll
              for (int n = 0; n < NP; ++n)
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                  const uint32_t w0 = t[g][jj][y & 2], w1 = t[g][jj][(y & 2) + 1];
                  // bytes y & 1 and 2 + (y & 1) as fp16: c + 16 c' of two positions
                  const uint32_t u0 = y & 1 ? __byte_perm(w0, 0, 0x4341) : w0 & 0x00ff00ffu;
                  const uint32_t u1 = y & 1 ? __byte_perm(w1, 0, 0x4341) : w1 & 0x00ff00ffu;
                  uint32_t a0, a1, a2, a3;
                  if constexpr (SPLIT) {
                    a0 = centre16((u0 << 4) & 0x00f000f0u);
                    a2 = centre16((u1 << 4) & 0x00f000f0u);
                    a1 = centre16(u0 & 0x00f000f0u);
                    a3 = centre16(u1 & 0x00f000f0u);
                  } else {
                    a0 = centre(u0, kMinus255);
                    a2 = centre(u1, kMinus255);
                    a1 = centre(u0 & 0x00f000f0u, kMinus240);
                    a3 = centre(u1 & 0x00f000f0u, kMinus240);
                  }
                  if (jj == 0) mma16_first(s[n][y], a0, a1, a2, a3, wv[g][jj][n][0], wv[g][jj][n][1]);
                  else mma16(s[n][y], a0, a1, a2, a3, wv[g][jj][n][0], wv[g][jj][n][1]);
                }
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              f32x2* om = o[i][4 * g + y];
              om[0] = add2(om[0], pack2(s[0][y][0], s[0][y][1]));
              om[1] = add2(om[1], pack2(s[0][y][2], s[0][y][3]));
              if constexpr (SPLIT) {
                const f32x2 low = pack2(1.f / kLow, 1.f / kLow);
                om[0] = fma2(pack2(s[NP - 1][y][0], s[NP - 1][y][1]), low, om[0]);
                om[1] = fma2(pack2(s[NP - 1][y][2], s[NP - 1][y][3]), low, om[1]);
              }
            }
          }
        }
      }
      __syncwarp();  // every lane has read the stage before its next copy is issued
    }

    // ---- the warps meet: numerators [slot][d] of each warp in its own ring
    const int busy = min(t1 - t0, kDecWarps);  // warps that had tiles, or would have had before they gave up a wait
    float* so = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      float ls, lz[NG], t;
      unpack2(lsum[i], ls, t);
      ls += t;
      ls += __shfl_xor_sync(0xffffffffu, ls, 1);
      ls += __shfl_xor_sync(0xffffffffu, ls, 2);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        unpack2(zsum[i][g], lz[g], t);
        lz[g] += t;
        lz[g] += __shfl_xor_sync(0xffffffffu, lz[g], 1);
        lz[g] += __shfl_xor_sync(0xffffffffu, lz[g], 2);
      }
      if (c4 == 0) {
        sm_m[warp][r8 + 8 * i] = mrun[i];
        sm_l[warp][r8 + 8 * i] = ls;
      }
      // slots 2 c4 and 2 c4 + 1 of the tile are this lane's columns
      float z0[NG], z1[NG], u0[NG], u1[NG];  // offsets' sums; 2^-shift
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        z0[g] = __shfl_sync(0xffffffffu, lz[g], 8 * c4);
        z1[g] = __shfl_sync(0xffffffffu, lz[g], 8 * c4 + 4);
        const float u = kWhole ? exp2_whole(-shift[i][g]) : ex2(-shift[i][g]);
        u0[g] = __shfl_sync(0xffffffffu, u, 8 * c4);
        u1[g] = __shfl_sync(0xffffffffu, u, 8 * c4 + 4);
      }
      if (warp < busy) {
#pragma unroll
        for (int m = 0; m < D / 16; ++m) {
          // rows r8: channel d (kPairs: plus 16 times channel d + 1); rows r8 + 8: 16 times channel d + 1
          const int d = 32 * (m / 2) + 4 * r8 + 2 * (m & 1);
          float e0, e1, h0, h1;
          unpack2(o[i][m][0], e0, e1);
          unpack2(o[i][m][1], h0, h1);
          if constexpr (kPairs) {
            e0 -= h0;
            e1 -= h1;
          }
          float* s0 = so + (8 * i + 2 * c4) * RP + d;
          *reinterpret_cast<float2*>(s0) =
              make_float2(fmaf(e0 * kUnitE, u0[m / 4], z0[m / 4]), fmaf(h0 * kUnitH, u0[m / 4], z0[m / 4]));
          *reinterpret_cast<float2*>(s0 + RP) =
              make_float2(fmaf(e1 * kUnitE, u1[m / 4], z1[m / 4]), fmaf(h1 * kUnitH, u1[m / 4], z1[m / 4]));
        }
      }
    }
    __syncthreads();
    if (threadIdx.x < kDecWarps * SLOTS) {
      const int w = threadIdx.x / SLOTS, s = threadIdx.x % SLOTS;
      float M = kNegInf;
#pragma unroll
      for (int x = 0; x < kDecWarps; ++x) M = fmaxf(M, sm_m[x][s]);
      const float m = sm_m[w][s];
      sm_f[w][s] = m == kNegInf ? 0.f : ex2(m - M);
    }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == ri.tiles;
    const int64_t part = ((int64_t)blockIdx.x * 2 + (t0 == 0 ? 1 : 0)) * SLOTS;
#pragma unroll 1
    for (int x = threadIdx.x * 4; x < SLOTS * D; x += kDecThreads * 4) {
      const int s = x / D, d = x % D;
      const int h = slot_head[s];
      if (h < 0) continue;
      float L = 0.f;
      float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int w = 0; w < busy; ++w) {
        const float f = sm_f[w][s];
        L = fmaf(sm_l[w][s], f, L);
        const float4 t =
            *reinterpret_cast<const float4*>(ring_all + (size_t)w * p.ring_bytes + (s * RP + d) * sizeof(float));
        O.x = fmaf(t.x, f, O.x);
        O.y = fmaf(t.y, f, O.y);
        O.z = fmaf(t.z, f, O.z);
        O.w = fmaf(t.w, f, O.w);
      }
      if (whole) {
        const float inv = L == 0.f ? 0.f : 1.f / L;
        const int64_t at = (int64_t)b * a.o_sb + (int64_t)h * a.o_sh + d;
        store_out(a.out, a.dtype, at, O.x * inv);
        store_out(a.out, a.dtype, at + 1, O.y * inv);
        store_out(a.out, a.dtype, at + 2, O.z * inv);
        store_out(a.out, a.dtype, at + 3, O.w * inv);
      } else {
        const int64_t rec = part + (h - grp.h0);
        *reinterpret_cast<float4*>(p.part_o + rec * D + d) = O;
        if (d == 0) {
          float M = kNegInf;
#pragma unroll
          for (int w = 0; w < kDecWarps; ++w) M = fmaxf(M, sm_m[w][s]);
          p.part_ml[rec * 2] = M;
          p.part_ml[rec * 2 + 1] = L;
        }
      }
    }
    fence_proxy_async_smem();  // the ring is written by bulk copies again
    __syncthreads();
    run = tile_base + t1;
  }
}

// Joins the partial results of items that CTA borders cut, and writes the zeros
// of rows without positions. One CTA per (request, query head): a warp takes
// every WARPS-th part, a lane four channels.
template <int D, int WARPS>
__global__ void __launch_bounds__(32 * WARPS) kv4_combine_kernel(const DecodePlan4 p, int grid, int slots) {
  constexpr int LPD = D / 4;            // lanes of a part
  constexpr int PPW = 32 / LPD;         // parts that a warp reads at a time
  __shared__ float sm_m[WARPS], sm_l[WARPS];
  __shared__ __align__(16) float sm_o[WARPS * PPW][D];
  const SagaKv4Args& a = p.a;
  const int b = blockIdx.x / a.Hq, h = blockIdx.x % a.Hq;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int G = a.Hq / a.pool.Hk, Gv = a.Hq / a.pool.Hv;
  const int kh = h / G, row = b * a.pool.Hk + kh;
  int sg = 0;
  SlotGroup grp = slot_group(kh, 0, G, Gv, slots, p.vheads);
  while (h >= grp.h0 + grp.n) grp = slot_group(kh, ++sg, G, Gv, slots, p.vheads);
  pdl_wait();
  if (threadIdx.x == 0 && a.lens[b] > a.max_pages * a.pool.page_len) set_status(a.status, SAGA_STATUS_PAGE_RANGE);
  const long long total = p.prefix[a.B * a.pool.Hk], first = p.prefix[row];
  const long long weight = divide(p.prefix[row + 1] - first, p.groups);
  const int64_t at = (int64_t)b * a.o_sb + (int64_t)h * a.o_sh;
  if (weight == 0) {
    for (int c = threadIdx.x; c < D; c += 32 * WARPS) store_out(a.out, a.dtype, at + c, 0.f);
    return;
  }
  const long long per = tiles_per_cta(total, grid);
  const long long begin = first + sg * weight + kItemTiles, end = first + (sg + 1) * weight;
  const int c0 = (int)divide(begin, per), n = (int)divide(end - 1, per) - c0 + 1;
  if (n == 1) return;  // one CTA had the whole item
  // part i: of CTA c0 + i; only the first part can begin with the item
  auto record = [&](int i) { return ((int64_t)(c0 + i) * 2 + (i == 0 ? 1 : 0)) * slots + (h - grp.h0); };
  const int sub = lane / LPD, d = (lane % LPD) * 4;
  // the first parts of each warp are on their way while the maximum is found
  constexpr int kEarly = 4;
  float4 early[kEarly];
#pragma unroll
  for (int j = 0; j < kEarly; ++j) {
    const int i = (warp + j * WARPS) * PPW + sub;
    if (i < n) early[j] = *reinterpret_cast<const float4*>(p.part_o + record(i) * D + d);
  }
  float m = kNegInf;
  for (int i = threadIdx.x; i < n; i += 32 * WARPS) m = fmaxf(m, p.part_ml[record(i) * 2]);
  m = warp_max(m);
  if (lane == 0) sm_m[warp] = m;
  __syncthreads();
  float M = sm_m[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) M = fmaxf(M, sm_m[w]);
  float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
  float L = 0.f;
  auto add = [&](int i, const float4& t) {
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + record(i) * 2);
    const float f = ml.x == kNegInf ? 0.f : ex2(ml.x - M);
    L = fmaf(ml.y, f, L);
    O.x = fmaf(t.x, f, O.x);
    O.y = fmaf(t.y, f, O.y);
    O.z = fmaf(t.z, f, O.z);
    O.w = fmaf(t.w, f, O.w);
  };
#pragma unroll
  for (int j = 0; j < kEarly; ++j) {
    const int i = (warp + j * WARPS) * PPW + sub;
    if (i < n) add(i, early[j]);
  }
#pragma unroll 4
  for (int i = (warp + kEarly * WARPS) * PPW + sub; i < n; i += WARPS * PPW)
    add(i, *reinterpret_cast<const float4*>(p.part_o + record(i) * D + d));
  *reinterpret_cast<float4*>(&sm_o[warp * PPW + sub][d]) = O;
  if (PPW == 2) L += __shfl_xor_sync(0xffffffffu, L, 16);
  if (lane == 0) sm_l[warp] = L;
  __syncthreads();
  for (int c = threadIdx.x; c < D; c += 32 * WARPS) {
    float o = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) l += sm_l[w];
#pragma unroll
    for (int w = 0; w < WARPS * PPW; ++w) o += sm_o[w][c];
    store_out(a.out, a.dtype, at + c, l == 0.f ? 0.f : o / l);
  }
}

// Sizes that follow from the shapes alone.
struct DecodeSizes {
  int nt, slots, groups, vheads, stages, ring_bytes, grid;
  size_t off_o, off_ml, total;
};

DecodeSizes decode_sizes(const SagaKv4Args& a) {
  DecodeSizes z;
  const int D = a.pool.D, G = a.Hq / a.pool.Hk, Gv = a.Hq / a.pool.Hv;
  const bool split = a.dtype == SAGA_FP32;
  // fp32 keeps two terms of every operand, which leaves registers for eight slots
  z.nt = G <= 8 || split ? 1 : 2;
  z.slots = 8 * z.nt;
  const int tile = kv4_tile_bytes(D);
  // Value heads per stage: two stages of five (nine) tiles fit a warp's ring. The cuts are the
  // same with the greatest number that occurs as the limit, so that sizes the stages.
  const int cap = D == 128 ? 4 : 8;
  z.groups = 1;
  z.vheads = 1;
  for (int kh = 0; kh < a.pool.Hk; ++kh) {
    int n = 0;
    for (;; ++n) {
      const SlotGroup s = slot_group(kh, n, G, Gv, z.slots, cap);
      if (s.n == 0) break;
      z.vheads = std::max(z.vheads, (s.h0 + s.n - 1) / Gv - s.h0 / Gv + 1);
      if (s.h0 + s.n >= (kh + 1) * G) { ++n; break; }
    }
    z.groups = std::max(z.groups, n);
  }
  const int stage = (1 + z.vheads) * tile;
  z.stages = std::max(2, std::min(kMaxRing, kRingBytes / kDecWarps / stage));
  z.ring_bytes = std::max(z.stages * stage, (int)((z.slots * (D + 4) * sizeof(float) + 127) / 128 * 128));
  z.grid = sm_count();
  const size_t rows = (size_t)a.B * a.pool.Hk;
  z.off_o = ((rows + 1) * sizeof(long long) + 255) / 256 * 256;
  z.off_ml = z.off_o + (size_t)z.grid * 2 * z.slots * D * sizeof(float);
  z.total = z.off_ml + (size_t)z.grid * 2 * z.slots * 2 * sizeof(float);
  return z;
}

template <int D, int NT, bool SPLIT>
int launch(const DecodePlan4& p, const DecodeSizes& z, cudaStream_t st) {
  auto* fn = kv4_decode_kernel<D, NT, SPLIT>;
  const int smem = z.ring_bytes * kDecWarps;
  // the limit is an attribute of the function on a device; it only rises
  static thread_local int dev_of = -1, raised = 0;
  int dev = 0;
  cudaGetDevice(&dev);
  cudaError_t e;
  if (dev != dev_of || smem > raised) {
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes);
    if (e != cudaSuccess) return abi_fail(SAGA_ERR_CUDA, std::string("kv4_decode_kernel: ") + cudaGetErrorString(e));
    dev_of = dev;
    raised = kRingBytes;
  }
  if (int rc = kv4_launch("kv4_decode_kernel", fn, dim3(z.grid), kDecThreads, smem, st, p)) return rc;
  // few rows have many parts each (147 parts: 6.1 us with 16 warps, 7.5 us with 8); many rows have few, and
  // their CTAs' number counts (768 rows: 6.7 us with 8 warps, 12.5 us with 16)
  const int rows = p.a.B * p.a.Hq;
  return rows <= z.grid ? kv4_launch("kv4_combine_kernel", kv4_combine_kernel<D, 16>, dim3((unsigned)rows), 512, 0, st,
                                     p, z.grid, z.slots)
                        : kv4_launch("kv4_combine_kernel", kv4_combine_kernel<D, 4>, dim3((unsigned)rows), 128, 0, st,
                                     p, z.grid, z.slots);
}

}  // namespace

size_t kv4_decode_workspace(const SagaKv4Args& a) { return decode_sizes(a).total; }

int launch_kv4_decode(const SagaKv4Args& a, cudaStream_t st) {
  const DecodeSizes z = decode_sizes(a);
  DecodePlan4 p;
  p.a = a;
  p.groups = z.groups;
  p.vheads = z.vheads;
  p.stages = z.stages;
  p.ring_bytes = z.ring_bytes;
  p.tpp_shift = 0;
  while ((kKv4Tile << p.tpp_shift) < a.pool.page_len) ++p.tpp_shift;
  uint8_t* ws = reinterpret_cast<uint8_t*>(a.workspace);
  p.prefix = reinterpret_cast<long long*>(ws);
  p.part_o = reinterpret_cast<float*>(ws + z.off_o);
  p.part_ml = reinterpret_cast<float*>(ws + z.off_ml);
  if (a.dtype == SAGA_FP32) return a.pool.D == 128 ? launch<128, 1, true>(p, z, st) : launch<64, 1, true>(p, z, st);
  if (z.nt == 1) return a.pool.D == 128 ? launch<128, 1, false>(p, z, st) : launch<64, 1, false>(p, z, st);
  return a.pool.D == 128 ? launch<128, 2, false>(p, z, st) : launch<64, 2, false>(p, z, st);
}

}  // namespace saga
