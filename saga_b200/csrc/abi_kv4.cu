// extern "C" entry points of the 4-bit paged cache operators: validation on
// the host, then the launchers.
#include <cmath>
#include <new>
#include <string>

#include "kv4.h"

namespace {

using saga::abi_begin;
using saga::abi_fail;

bool is_fp(int dt) { return dt == SAGA_BF16 || dt == SAGA_FP16 || dt == SAGA_FP32; }
bool aligned(const void* p, int a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
int invalid(const char* m) { return abi_fail(SAGA_ERR_INVALID, m); }

int check_geometry(int32_t D, int32_t page_len) {
  if (D != 64 && D != 128) return abi_fail(SAGA_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
  if (page_len < 32 || (page_len & (page_len - 1)))
    return invalid("page_len must be a power of two and at least 32");
  return SAGA_OK;
}

int check_pool(const SagaKv4Pool& p) {
  if (int rc = check_geometry(p.D, p.page_len)) return rc;
  if (p.Hk <= 0 || p.Hv <= 0 || p.num_pages <= 0) return invalid("Hk, Hv and num_pages must be positive");
  if ((int64_t)p.num_pages * (p.page_len / saga::kKv4Tile) > 0x7fffffffll)
    return abi_fail(SAGA_ERR_UNSUPPORTED, "the pool has more than 2^31 tiles");
  if (!p.k || !p.v || !aligned(p.k, 16) || !aligned(p.v, 16))
    return invalid("the pool's keys and values must be non-NULL and 16-byte aligned");
  if ((p.k_lo == nullptr) != (p.k_hi == nullptr)) return invalid("k_lo and k_hi go together");
  if (!aligned(p.k_lo, 16) || !aligned(p.k_hi, 16)) return invalid("the key bounds must be 16-byte aligned");
  return SAGA_OK;
}

int check_table(const void* table, int64_t pt_sb, int32_t max_pages, int32_t page_len) {
  if (!table || !aligned(table, 4)) return invalid("page_table must be non-NULL and 4-byte aligned");
  if (max_pages <= 0 || pt_sb < max_pages) return invalid("page table rows must hold max_pages > 0 entries");
  if ((int64_t)max_pages * page_len > 0x7fffffffll - 64)
    return abi_fail(SAGA_ERR_UNSUPPORTED, "a page table row covers more than 2^31 positions");
  return SAGA_OK;
}

// Shapes alone (enough for a workspace query).
int check_shapes(const SagaKv4Args* a, int op) {
  if (!a) return invalid("args is NULL");
  if (int rc = check_geometry(a->pool.D, a->pool.page_len)) return rc;
  if (!is_fp(a->dtype)) return invalid("dtype must be bf16, fp16 or fp32");
  if (a->B < 0 || a->Hq <= 0 || a->pool.Hk <= 0 || a->pool.Hv <= 0)
    return invalid("B >= 0, Hq, Hk, Hv > 0 required");
  if (a->Hq % a->pool.Hk) return invalid("Hq must be a multiple of Hk");
  if (a->Hq % a->pool.Hv) return invalid("Hq must be a multiple of Hv");
  if ((int64_t)a->B * a->Hq > 0x7fffffffll || (int64_t)a->B * a->pool.Hk > 0x7fffff00ll)
    return abi_fail(SAGA_ERR_UNSUPPORTED, "too many (request, query head) rows");
  if (a->max_pages <= 0) return invalid("max_pages must be positive");
  if (op == SAGA_KV4_SELECT || a->blocks) {
    if (a->top <= 0) return invalid("top must be positive");
    if ((int64_t)a->top * a->pool.page_len > 0x7fffffffll - 64)
      return abi_fail(SAGA_ERR_UNSUPPORTED, "the blocks cover more than 2^31 positions");
  }
  return SAGA_OK;
}

int check_call(const SagaKv4Args* a, int op) {
  if (int rc = check_shapes(a, op)) return rc;
  if (int rc = check_pool(a->pool)) return rc;
  if (a->B == 0) return SAGA_OK;
  if (int rc = check_table(a->page_table, a->pt_sb, a->max_pages, a->pool.page_len)) return rc;
  if (!a->q) return invalid("q must be non-NULL");
  if (!a->lens) return invalid("lens must be non-NULL");
  if (op == SAGA_KV4_DECODE) {
    if (!a->out) return invalid("out must be non-NULL");
    if (!std::isfinite(a->scaling)) return invalid("scaling must be finite");
    if ((a->blocks == nullptr) != (a->counts == nullptr)) return invalid("blocks and counts go together");
  } else {
    if (!a->pool.k_lo) return invalid("select needs the pool's key bounds");
    if (!a->blocks || !a->counts) return invalid("blocks and counts must be non-NULL");
    if (a->keep_first < 0 || a->keep_last < 1) return invalid("keep_first >= 0 and keep_last >= 1 required");
    if ((int64_t)a->keep_first + a->keep_last > a->top) return invalid("top must cover keep_first + keep_last");
  }
  return SAGA_OK;
}

// Exceptions of the standard library (a failed allocation) must not cross the C boundary.
template <class F>
int guarded(F f) {
  try {
    abi_begin();
    return f();
  } catch (...) {
    return SAGA_ERR_CUDA;
  }
}

int run(const SagaKv4Args* a, int op, void* stream) {
  if (int rc = check_call(a, op)) return rc;
  if (a->B == 0) return SAGA_OK;
  const size_t need = op == SAGA_KV4_DECODE ? saga::kv4_decode_workspace(*a) : saga::kv4_select_workspace(*a);
  if (!a->workspace || !aligned(a->workspace, 16) || a->workspace_bytes < need)
    return abi_fail(SAGA_ERR_WORKSPACE, "workspace missing, not 16-byte aligned or smaller than saga_kv4_workspace_bytes");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return op == SAGA_KV4_DECODE ? saga::launch_kv4_decode(*a, st) : saga::launch_kv4_select(*a, st);
}

int check_rows(const SagaKv4Pool* p, int dtype, int64_t T, const void* k, const void* v, const int64_t* slots) {
  if (!p) return invalid("pool is NULL");
  if (int rc = check_pool(*p)) return rc;
  if (!is_fp(dtype)) return invalid("dtype must be bf16, fp16 or fp32");
  if (T < 0) return invalid("T must not be negative");
  if (T > 0 && (!k || !v || !slots)) return invalid("k, v and slots must be non-NULL");
  if (T * (int64_t)(p->Hk > p->Hv ? p->Hk : p->Hv) > (1ll << 40)) return invalid("too many rows");
  return SAGA_OK;
}

}  // namespace

namespace saga {
int sm_count() {
  static thread_local int dev_of = -1, sms = 0;
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev != dev_of) {
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    dev_of = dev;
  }
  return sms > 0 ? sms : 148;
}
}  // namespace saga

extern "C" {

size_t saga_kv4_page_bytes(int32_t D, int32_t page_len) {
  return guarded([&] { return check_geometry(D, page_len); }) ? 0
                                                              : (size_t)page_len / saga::kKv4Tile *
                                                                    saga::kv4_tile_bytes(D);
}

int saga_kv4_write(const SagaKv4Pool* pool, int32_t dtype, int64_t T, const void* k, int64_t k_st, int64_t k_sh,
                   const void* v, int64_t v_st, int64_t v_sh, const int64_t* slots, int32_t* status, void* stream) {
  return guarded([&]() -> int {
    if (int rc = check_rows(pool, dtype, T, k, v, slots)) return rc;
    if (T == 0) return SAGA_OK;
    return saga::launch_kv4_write(*pool, dtype, T, k, k_st, k_sh, v, v_st, v_sh, slots, status,
                                  reinterpret_cast<cudaStream_t>(stream));
  });
}

int saga_kv4_read(const SagaKv4Pool* pool, int32_t dtype, int64_t T, const int64_t* slots, void* k, int64_t k_st,
                  int64_t k_sh, void* v, int64_t v_st, int64_t v_sh, int32_t* status, void* stream) {
  return guarded([&]() -> int {
    if (int rc = check_rows(pool, dtype, T, k, v, slots)) return rc;
    if (T == 0) return SAGA_OK;
    return saga::launch_kv4_read(*pool, dtype, T, slots, k, k_st, k_sh, v, v_st, v_sh, status,
                                 reinterpret_cast<cudaStream_t>(stream));
  });
}

size_t saga_kv4_workspace_bytes(const SagaKv4Args* args, int32_t op) {
  size_t n = 0;
  const int rc = guarded([&]() -> int {
    if (op != SAGA_KV4_DECODE && op != SAGA_KV4_SELECT) return invalid("unknown op");
    if (int e = check_shapes(args, op)) return e;
    n = op == SAGA_KV4_DECODE ? saga::kv4_decode_workspace(*args) : saga::kv4_select_workspace(*args);
    return SAGA_OK;
  });
  return rc ? 0 : n;
}

int saga_kv4_decode(const SagaKv4Args* args, void* stream) {
  return guarded([&] { return run(args, SAGA_KV4_DECODE, stream); });
}

int saga_kv4_select(const SagaKv4Args* args, void* stream) {
  return guarded([&] { return run(args, SAGA_KV4_SELECT, stream); });
}

int saga_page_tables(const SagaPageTableArgs* a, void* stream) {
  return guarded([&]() -> int {
    if (!a) return invalid("args is NULL");
    if (a->page_len < 32 || (a->page_len & (a->page_len - 1)))
      return invalid("page_len must be a power of two and at least 32");
    if (a->B < 0 || a->num_tokens < 0 || a->num_tokens > 0x7fffffffll)
      return invalid("B >= 0 and 0 <= num_tokens < 2^31 required");
    if (!a->offsets || !a->free_state || !a->free_state_out) return invalid("offsets and free states must be non-NULL");
    if (a->num_tokens && (!a->slots || !a->positions)) return invalid("slots and positions must be non-NULL");
    if (a->ring < 0 || (a->ring && !a->free_pages)) return invalid("free_pages must hold `ring` entries");
    if (a->B) {
      if (int rc = check_table(a->page_table, a->pt_sb, a->max_pages, a->page_len)) return rc;
      if (!a->lens || !a->new_lens || !a->lens_out) return invalid("lens, new_lens and lens_out must be non-NULL");
      if (!a->workspace || !aligned(a->workspace, 16) || a->workspace_bytes < 16 * (size_t)a->B)
        return abi_fail(SAGA_ERR_WORKSPACE, "a 16-byte aligned workspace of 16 * B bytes is required");
    }
    return saga::launch_page_tables(*a, reinterpret_cast<cudaStream_t>(stream));
  });
}

int saga_slot_map(int32_t B, int32_t page_len, const int32_t* page_table, int64_t pt_sb, int32_t max_pages,
                  const int32_t* starts, const int32_t* lens, int64_t num_tokens, int64_t* slots, int32_t* offsets,
                  int32_t* status, void* stream) {
  return guarded([&]() -> int {
    if (page_len < 32 || (page_len & (page_len - 1)))
      return invalid("page_len must be a power of two and at least 32");
    if (B < 0 || num_tokens < 0 || num_tokens > 0x7fffffffll)
      return invalid("B >= 0 and 0 <= num_tokens < 2^31 required");
    if (!offsets || (num_tokens && !slots)) return invalid("slots and offsets must be non-NULL");
    if (B) {
      if (int rc = check_table(page_table, pt_sb, max_pages, page_len)) return rc;
      if (!lens) return invalid("lens must be non-NULL");
    }
    return saga::launch_slot_map(B, page_len, page_table, pt_sb, max_pages, starts, lens, num_tokens, slots, offsets,
                                 status, reinterpret_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
