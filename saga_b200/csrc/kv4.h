// Host launchers of the 4-bit paged cache operators (internal).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <string>

#include "../../include/saga_b200.h"

namespace saga {

// abi.cu: error text and launch record of the calling thread.
int abi_fail(int code, const std::string& msg);
void abi_begin();
void abi_launched(const char* name);

constexpr int kKv4Tile = 32;  // positions of a tile: its codes and its scales are contiguous

__host__ __device__ constexpr int kv4_tile_bytes(int D) { return kKv4Tile * (D / 2 + D / 16); }

int launch_kv4_write(const SagaKv4Pool& p, int dt, int64_t T, const void* k, int64_t k_st, int64_t k_sh,
                     const void* v, int64_t v_st, int64_t v_sh, const int64_t* slots, int* status, cudaStream_t st);
int launch_kv4_read(const SagaKv4Pool& p, int dt, int64_t T, const int64_t* slots, void* k, int64_t k_st,
                    int64_t k_sh, void* v, int64_t v_st, int64_t v_sh, int* status, cudaStream_t st);
size_t kv4_decode_workspace(const SagaKv4Args& a);
int launch_kv4_decode(const SagaKv4Args& a, cudaStream_t st);
size_t kv4_select_workspace(const SagaKv4Args& a);
int launch_kv4_select(const SagaKv4Args& a, cudaStream_t st);
int launch_page_tables(const SagaPageTableArgs& a, cudaStream_t st);
int launch_slot_map(int B, int page_len, const int32_t* pt, int64_t pt_sb, int max_pages, const int32_t* starts,
                    const int32_t* lens, int64_t T, int64_t* slots, int32_t* offsets, int* status, cudaStream_t st);

// SAGA_OK, or SAGA_ERR_CUDA with the launch's error.
inline int kv4_launched(const char* name) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return abi_fail(SAGA_ERR_CUDA, std::string(name) + ": " + cudaGetErrorString(e));
  abi_launched(name);
  return SAGA_OK;
}

}  // namespace saga
