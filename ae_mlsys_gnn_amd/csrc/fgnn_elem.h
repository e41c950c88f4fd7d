// Element types of the dense operators (rows of fp32, bf16, fp16 and 8-bit values): sizes, 16-byte vectors, conversions.
#pragma once
#include "fgnn_common.h"

typedef int8_t fe_i8;
struct fe_e4m3 { uint8_t bits; };           // 1-4-3, bias 7, no infinities, 448 the largest

// 16 bytes of elements that start at any element: the hardware takes 128-bit loads and stores at any byte address.
template <typename T> struct fe_vec { typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T)))); };
template <typename T> constexpr int fe_width = 16 / sizeof(T);

static inline int fe_size(int type) { return type == FGNN_F32 ? 4 : type == FGNN_BF16 || type == FGNN_F16 ? 2 : 1; }
template <int TYPE> constexpr int fe_size_of = TYPE == FGNN_F32 ? 4 : TYPE == FGNN_BF16 || TYPE == FGNN_F16 ? 2 : 1;
static inline bool fe_is_float(int type) { return type == FGNN_F32 || type == FGNN_BF16 || type == FGNN_F16; }
static inline bool fe_is_eight(int type) { return type == FGNN_I8 || type == FGNN_E4M3; }
// The largest value that rows are scaled to in 8 bits.
static inline float fe_top(int type) { return type == FGNN_I8 ? 127.f : 448.f; }

// An element of a type known at run time, for the few values a kernel reads once (weights, bias).
__device__ __forceinline__ float fe_load(const void *p, int64_t i, int type)
{
    return type == FGNN_F32 ? ((const float *)p)[i] : type == FGNN_BF16 ? (float)((const __bf16 *)p)[i] : (float)((const _Float16 *)p)[i];
}
__device__ __forceinline__ void fe_store(void *p, int64_t i, int type, float v)
{
    if (type == FGNN_F32) ((float *)p)[i] = v;
    else if (type == FGNN_BF16) ((__bf16 *)p)[i] = (__bf16)v;
    else ((_Float16 *)p)[i] = (_Float16)v;
}

// Calls f.template operator()<T>() for a floating type.
template <typename Fn>
static inline void fe_dispatch(int type, Fn &&f)
{
    if (type == FGNN_F32) f.template operator()<float>();
    else if (type == FGNN_BF16) f.template operator()<__bf16>();
    else f.template operator()<_Float16>();
}

// out [cols], of a floating type = the column sums of part [rows, cols], added in a fixed order (fgnn_norm.hip).
int fgnn_sum_parts(const float *part, int rows, int cols, void *out, int type, hipStream_t st);
