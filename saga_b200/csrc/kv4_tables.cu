// Block tables and slot maps of a step, built on the GPU from the requests'
// lengths. The sums over the requests are one CTA's scan; the tokens and the
// returned pages are then independent of one another.
//
// There is next to nothing to move (12 bytes per token), so latency is all: the
// scan takes 5.6 us for 512 requests, the tokens 9.4 us for 65,536 of them from
// cold caches (offsets, request, table entry: loads that follow one another).
#include "kv4.cuh"

namespace saga {

namespace {

constexpr int kScan = 1024;  // threads of the scanning CTA

// Per request, for the token phase (the 16 bytes per request of the workspace).
struct TableRow {
  int len;    // positions held before the step; -1: no new tokens are placed
  int first;  // index in the ring of the request's first new page
  int back;   // index in the ring of the first page that the request returns; -1: none
  int held;   // pages held before the step
};

// Exclusive sums over the CTA's threads of N values; totals in tot.
template <int N>
__device__ __forceinline__ void scan(long long (&v)[N], long long (&tot)[N], long long (*sm)[33]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long inc[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    long long x = v[j];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    inc[j] = x;
    if (lane == 31) sm[j][warp] = x;
  }
  __syncthreads();
  if (warp < N) {
    const long long own = sm[warp][lane];
    long long x = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncwarp();
    sm[warp][lane] = x - own;
    if (lane == 31) sm[warp][32] = x;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < N; ++j) {
    tot[j] = sm[j][32];
    v[j] = sm[j][warp] + inc[j] - v[j];
  }
  __syncthreads();
}

__device__ void table_scan(const SagaPageTableArgs& a, TableRow* rows) {
  __shared__ long long sm[2][33];
  __shared__ int taken_sm, returned_sm;
  if (threadIdx.x == 0) taken_sm = returned_sm = 0;
  const int shift = __ffs(a.page_len) - 1;
  const long long cover = (long long)a.max_pages << shift;
  const int head = a.free_state[0];
  const int count = min(max(a.free_state[1], 0), a.ring);
  const int h0 = a.ring ? (int)((unsigned)max(head, 0) % (unsigned)a.ring) : 0;
  long long tok = 0, want = 0, ret = 0;
  for (int base = 0; base < a.B; base += kScan) {
    const int b = base + threadIdx.x;
    const bool in = b < a.B;
    const int len = in ? max(a.lens[b], 0) : 0;
    const int raw = in ? a.new_lens[b] : 0;
    const int add = max(raw, 0);
    const long long end = (long long)len + add;
    const int held = (int)(((long long)len + a.page_len - 1) >> shift);
    long long v1[1] = {add}, tot1[1];
    scan(v1, tot1, sm);
    const long long start = tok + v1[0];
    tok += tot1[0];
    const bool fits = end <= cover && start + add <= a.num_tokens;
    const int need = fits ? (int)(((end + a.page_len - 1) >> shift) - held) : 0;
    const int back = in && raw < 0 ? min(held, a.max_pages) : 0;
    long long v[2] = {need, back}, tot[2];
    scan(v, tot, sm);
    const long long upto = want + v[0] + need;
    const bool granted = fits && (need == 0 || upto <= count);
    // pages go back to the entries that are not free, so nothing that is free is written over
    const long long before = ret + v[1];
    const bool room = back == 0 || before + back <= a.ring - count;
    want += tot[0];
    ret += tot[1];
    // the granted requests that need pages are the first ones that do, so the last one's sum is the total; the
    // same holds of the returned pages
    if (granted && need) atomicMax(&taken_sm, (int)upto);
    if (room && back) atomicMax(&returned_sm, (int)(before + back));
    if (in) {
      TableRow r;
      r.len = granted ? len : -1;
      r.first = a.ring ? (int)((h0 + upto - need) % a.ring) : 0;
      r.back = back && room ? (int)((h0 + (long long)count + before) % a.ring) : -1;
      r.held = held;
      rows[b] = r;
      a.offsets[b + 1] = (int)min(start + add, 0x7fffffffll);
      a.lens_out[b] = raw < 0 ? (room ? 0 : len) : granted ? (int)end : len;
      if (!granted && add > 0) set_status(a.status, SAGA_STATUS_OUT_OF_PAGES);
      if (!room) set_status(a.status, SAGA_STATUS_PAGE_RANGE);
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    const int taken = taken_sm;
    a.offsets[0] = 0;
    a.free_state_out[0] = a.ring ? (int)((h0 + taken) % a.ring) : 0;
    a.free_state_out[1] = count - taken + returned_sm;
  }
}

constexpr int kShared = 2048;  // offsets kept in shared memory (a bisection in global memory waits at every step)

// Copies the offsets to shared memory if they fit; returns where to read them.
__device__ __forceinline__ const int32_t* stage_offsets(const int32_t* offsets, int B, int32_t* sm) {
  if (B >= kShared) return offsets;
  for (int i = threadIdx.x; i <= B; i += blockDim.x) sm[i] = offsets[i];
  __syncthreads();
  return sm;
}
// The request that row i belongs to: offsets[lo] <= i < offsets[lo + 1].
__device__ __forceinline__ int find_request(const int32_t* offsets, int B, int64_t i) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (offsets[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Token `i`: its request, slot and position; the first token of a new page also
// writes the page table's entry.
__device__ __forceinline__ void table_token(const SagaPageTableArgs& a, const TableRow* rows, const int32_t* offsets,
                                            int64_t i) {
  int64_t slot = -1;
  int pos = 0;
  if (a.B > 0 && i < offsets[a.B]) {
    const int lo = find_request(offsets, a.B, i);
    const TableRow r = rows[lo];
    if (r.len >= 0) {
      pos = r.len + (int)(i - offsets[lo]);
      const int shift = __ffs(a.page_len) - 1;
      const int p = pos >> shift, off = pos & (a.page_len - 1);
      int32_t* entry = a.page_table + (int64_t)lo * a.pt_sb + p;
      int page;
      if (p < r.held) {
        page = *entry;
      } else {
        page = a.free_pages[((unsigned)r.first + (unsigned)(p - r.held)) % (unsigned)a.ring];
        if (off == 0) *entry = page;
      }
      slot = (int64_t)page * a.page_len + off;
    }
  }
  a.slots[i] = slot;
  a.positions[i] = pos;
}

// A warp returns the pages of request b to the ring.
__device__ __forceinline__ void table_return(const SagaPageTableArgs& a, const TableRow* rows, int b) {
  const TableRow r = rows[b];
  if (r.back < 0) return;
  for (int j = threadIdx.x & 31; j < min(r.held, a.max_pages); j += 32)
    a.free_pages[((unsigned)r.back + (unsigned)j) % (unsigned)a.ring] = a.page_table[(int64_t)b * a.pt_sb + j];
}

__global__ void __launch_bounds__(kScan) page_tables_scan_kernel(SagaPageTableArgs a, bool all) {
  pdl_wait();
  TableRow* rows = reinterpret_cast<TableRow*>(a.workspace);
  table_scan(a, rows);
  if (!all) return;
  __shared__ int32_t off_sm[kShared + 1];
  __syncthreads();
  const int32_t* offsets = stage_offsets(a.offsets, a.B, off_sm);
  for (int64_t i = threadIdx.x; i < a.num_tokens; i += kScan) table_token(a, rows, offsets, i);
  for (int b = threadIdx.x >> 5; b < a.B; b += kScan / 32) table_return(a, rows, b);
}

__global__ void __launch_bounds__(256) page_tables_token_kernel(SagaPageTableArgs a) {
  pdl_wait();
  const TableRow* rows = reinterpret_cast<const TableRow*>(a.workspace);
  __shared__ int32_t off_sm[kShared + 1];
  const int32_t* offsets = stage_offsets(a.offsets, a.B, off_sm);
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < a.num_tokens) table_token(a, rows, offsets, i);
  for (int b = (int)(i >> 5); b < a.B; b += (int)gridDim.x * 8) table_return(a, rows, b);
}

__global__ void __launch_bounds__(kScan) slot_offsets_kernel(int B, int64_t cover, const int32_t* starts,
                                                             const int32_t* lens, int32_t* offsets, int* status) {
  __shared__ long long sm[1][33];
  pdl_wait();
  long long tok = 0;
  for (int base = 0; base < B; base += kScan) {
    const int b = base + threadIdx.x;
    long long n = 0;
    if (b < B) {
      long long end = lens[b];
      if (end > cover) {
        set_status(status, SAGA_STATUS_PAGE_RANGE);
        end = cover;
      }
      n = max(end - max(starts ? starts[b] : 0, 0), 0ll);
    }
    long long v[1] = {n}, tot[1];
    scan(v, tot, sm);
    if (b < B) offsets[b + 1] = (int)min(tok + v[0] + n, 0x7fffffffll);
    tok += tot[0];
  }
  if (threadIdx.x == 0) offsets[0] = 0;
}

__global__ void __launch_bounds__(256) slot_map_kernel(int B, int page_len, const int32_t* pt, int64_t pt_sb,
                                                       const int32_t* starts, int64_t T_, int64_t* slots,
                                                       const int32_t* offsets) {
  pdl_wait();
  __shared__ int32_t off_sm[kShared + 1];
  offsets = stage_offsets(offsets, B, off_sm);
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= T_) return;
  int64_t slot = -1;
  if (B > 0 && i < offsets[B]) {
    const int lo = find_request(offsets, B, i);
    const int pos = max(starts ? starts[lo] : 0, 0) + (int)(i - offsets[lo]);
    const int shift = __ffs(page_len) - 1;
    slot = (int64_t)pt[(int64_t)lo * pt_sb + (pos >> shift)] * page_len + (pos & (page_len - 1));
  }
  slots[i] = slot;
}

}  // namespace

int launch_page_tables(const SagaPageTableArgs& a, cudaStream_t st) {
  // few tokens are left to the scanning CTA: 64 requests with 1024 tokens take 5.5 us by one launch, 6.0 us by
  // two; with 2048 tokens 6.4 us and 5.8 us
  const bool all = a.num_tokens <= 1024;
  int rc = kv4_launch("page_tables_scan_kernel", page_tables_scan_kernel, dim3(1), kScan, 0, st, a, all);
  if (rc || all) return rc;
  return kv4_launch("page_tables_token_kernel", page_tables_token_kernel,
                    dim3((unsigned)((a.num_tokens + 255) / 256)), 256, 0, st, a);
}

int launch_slot_map(int B, int page_len, const int32_t* pt, int64_t pt_sb, int max_pages, const int32_t* starts,
                    const int32_t* lens, int64_t T, int64_t* slots, int32_t* offsets, int* status, cudaStream_t st) {
  int rc = kv4_launch("slot_offsets_kernel", slot_offsets_kernel, dim3(1), kScan, 0, st, B,
                      (int64_t)max_pages * page_len, starts, lens, offsets, status);
  if (rc || T == 0) return rc;
  return kv4_launch("slot_map_kernel", slot_map_kernel, dim3((unsigned)((T + 255) / 256)), 256, 0, st, B, page_len, pt,
                    pt_sb, starts, T, slots, offsets);
}

}  // namespace saga
