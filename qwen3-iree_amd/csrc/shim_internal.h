// Internal interface between the C-ABI shim (q8gemv_shim.cpp), the cache
// operators (cache_shim.cpp) and the allocation-free entry point
// (q8gemv_noalloc.hip); not part of the ABI.
#ifndef QWEN3_SHIM_INTERNAL_H
#define QWEN3_SHIM_INTERNAL_H

#include <hip/hip_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

struct f16_cache;

namespace q8_shim {

// Sets the calling thread's error message (q8gemv_last_error) and returns code.
int error(int code, const char* msg);
int hip_error(hipError_t e, const char* what);

// Q8_OK once q8gemv_init has run.
int ready();
int compute_units();
// The launches every entry point makes (1-D and 3-D grids of 1-D workgroups).
int launch(hipFunction_t fn, uint32_t grid, uint32_t block, void** args, hipStream_t stream);
int launch3(hipFunction_t fn, uint32_t gx, uint32_t gy, uint32_t gz, uint32_t block, void** args,
            hipStream_t stream);

// Implemented in cache_shim.cpp: loads the code object at `path` (a failure
// leaves the cache operators reporting Q8_ERR_CODE_OBJECT) and unloads it.
void cache_load(const char* path);
void cache_unload();
// The workspace bytes of this one call of f16_attn_tree (arguments in range), at most
// f16_attn_tree_workspace_bytes.
size_t attn_tree_need(const f16_cache* cache, int32_t len, int32_t n, int32_t q_heads);
// The RoPE table of a tree's nodes (tree_rope_k).
int tree_rope(const int32_t* depth, int32_t position, int32_t n, void* table, hipStream_t stream);

// Q8_OK once q8gemv_init has run and the allocation-free scratch of its
// device was set up; otherwise the status and message of what is missing.
int noalloc_ready();

// Argument checks of f16_gemv_argmax_rows other than the workspace.
int validate_f16_argmax(const void* w_f16, int64_t n_rows, const void* x_f16,
                        const void* logits_f16, const int32_t* token);

// The vocab GEMV + argmax and its finalize on `s`, the argmax key at
// `workspace` (a device address: 16-byte aligned, zero before the launch,
// zero again after the finalize).
int launch_f16_argmax(const void* w_f16, int64_t n_rows, const void* x_f16, void* logits_f16,
                      int32_t* token, void* workspace, hipStream_t s);

// Implemented in q8gemv_noalloc.hip: looks up the scratch array's address on
// `device` (which must be current) and zero-fills it; called by q8gemv_init.
int noalloc_setup(int device);

}  // namespace q8_shim

#endif
