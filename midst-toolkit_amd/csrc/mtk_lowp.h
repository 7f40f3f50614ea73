// mtk_lowp.h — element types and vector access shared by the row routing, low-rank adapter and AdamW kernels.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "mtk_common.h"

typedef _Float16 mtk_f16;
typedef __bf16 mtk_bf16;

// Elements per 16-byte piece, and a piece whose address need only be a multiple of the element's size: rows of odd widths start
// anywhere, and gfx950 loads and stores 16 bytes at any address (one instruction; a piece that straddles a cache line costs a second
// line access).  May_alias: the same memory is read as T elsewhere.
template <typename T> struct mtk_piece { static constexpr int n = 16 / sizeof(T); };
template <typename T> struct __attribute__((packed, aligned(alignof(T)), may_alias)) mtk_vec { T v[16 / sizeof(T)]; };

template <typename T> __device__ __forceinline__ mtk_vec<T> mtk_ld(const T* p) { return *reinterpret_cast<const mtk_vec<T>*>(p); }
template <typename T> __device__ __forceinline__ void mtk_st(T* p, const mtk_vec<T>& v) { *reinterpret_cast<mtk_vec<T>*>(p) = v; }
// past the caches, both ways
template <typename T> __device__ __forceinline__ void mtk_st_nt(T* p, const mtk_vec<T>& v) {
    typedef uint32_t words __attribute__((ext_vector_type(4), aligned(2)));  // see mtk_vec
    __builtin_nontemporal_store(__builtin_bit_cast(words, v), reinterpret_cast<words*>(p));
}
template <typename T> __device__ __forceinline__ mtk_vec<T> mtk_ld_nt(const T* p) {
    typedef uint32_t words __attribute__((ext_vector_type(4), aligned(2)));
    return __builtin_bit_cast(mtk_vec<T>, __builtin_nontemporal_load(reinterpret_cast<const words*>(p)));
}
// the first `n` elements of a piece, zeros behind them
template <typename T> __device__ __forceinline__ mtk_vec<T> mtk_ld_n(const T* p, int n) {
    mtk_vec<T> v;
#pragma unroll
    for (int i = 0; i < mtk_piece<T>::n; ++i) v.v[i] = i < n ? p[i] : T(0);
    return v;
}
template <typename T> __device__ __forceinline__ void mtk_st_n(T* p, const mtk_vec<T>& v, int n) {
#pragma unroll
    for (int i = 0; i < mtk_piece<T>::n; ++i)
        if (i < n) p[i] = v.v[i];
}

// runs f with a value of the C type that `dtype` (enum mtk_dtype) names; the caller has checked it
template <typename F> static inline void mtk_by_type(int dtype, F f) {
    if (dtype == MTK_DT_F32) f(float(0));
    else if (dtype == MTK_DT_BF16) f(mtk_bf16(0));
    else f(mtk_f16(0));
}
static inline bool mtk_dtype_ok(int dtype) { return dtype >= MTK_DT_F32 && dtype <= MTK_DT_F16; }
static inline int mtk_dtype_size(int dtype) { return dtype == MTK_DT_F32 ? 4 : 2; }
__host__ __device__ static inline int64_t mtk_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
