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

int sm_count();  // of the current device

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

// Launches a kernel that may start while the one before it in the stream is
// still running. Every kernel launched so begins with pdl_wait() (kv4.cuh),
// before it touches memory: what comes before it in the stream has then
// finished, whether or not it was launched this way.
template <class... P, class... A>
int kv4_launch(const char* name, void (*fn)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t st,
               A... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, static_cast<P>(args)...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return abi_fail(SAGA_ERR_CUDA, std::string(name) + ": " + cudaGetErrorString(e));
  }
  abi_launched(name);
  return SAGA_OK;
}

}  // namespace saga
