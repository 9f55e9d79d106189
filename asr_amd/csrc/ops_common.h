// Shared by the operators on device memory (ops_rows.hip, ops_attention.hip; include/asr_amd.h "operators on device memory").
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "../../include/asr_amd.h"

// Records the message that asr_ops_last_error() of this host thread returns; `code` is handed back.  Never throws.
int ops_fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
// ASR_OK, or ASR_ERR_HIP with the launch's error
int ops_launched(const char* what, hipError_t e);

// Queues a kernel that takes one argument struct and returns this launch's own status (not an error an earlier call left behind)
template <typename A> static inline hipError_t ops_launch(void (*kernel)(A), dim3 grid, dim3 block, hipStream_t s, A args)
{
    void* p[1] = {&args};
    return hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, p, 0, s);
}

static inline int64_t ops_dtype_size(int32_t dtype) { return dtype == ASR_F32 ? 4 : 2; }
static inline bool ops_dtype_ok(int32_t dtype) { return dtype == ASR_F32 || dtype == ASR_BF16 || dtype == ASR_F16; }
// rows of a [n, t, heads, d] array that start on 16 bytes: base and strides (one of a dimension of size 1 is never used)
static inline bool ops_rows16(const void* p, const int64_t* stride, int64_t n, int64_t t, int64_t heads, int32_t dtype)
{
    const int64_t per = 16 / ops_dtype_size(dtype);
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (n <= 1 || stride[0] % per == 0) && (t <= 1 || stride[1] % per == 0) &&
           (heads <= 1 || stride[2] % per == 0);
}

// the argument structs are packed by asr_amd/ops.py: their layout is fixed
static_assert(sizeof(asr_token_logprobs_args) == 6 * 8 + 2 * 8 + 4 * 4, "layout");
static_assert(sizeof(asr_cross_attention_args) == 7 * 8 + 14 * 8 + 8 * 4, "layout");
static_assert(sizeof(asr_kv8_append_args) == 8 * 8 + 8 * 8 + 6 * 4, "layout");
static_assert(sizeof(asr_kv8_attention_args) == 8 * 8 + 9 * 8 + 9 * 4 + 4, "layout");

// log p(token), entropy and top-k per row (ops_rows.hip); the engine's scoring path calls it on its float32 logits
int ops_token_logprobs(const asr_token_logprobs_args& a, hipStream_t s);
