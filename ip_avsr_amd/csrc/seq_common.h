// Shared by the sequence operators (layernorm.hip, causal_conv.hip, selective_scan.hip): (B, T, channels) views, vector loads in
// float32 / bfloat16, sums over lanes in registers, and the fixed-order sum of per-workgroup partial rows.
#pragma once
#include "adn_common.h"
#include <algorithm>

namespace adn {
namespace seq {

// element (b, t, c) of a tensor at p[b sb + t st + c]
template <typename T> struct View {
    T* p;
    int64_t sb, st;
    __device__ __forceinline__ T* row(int b, int t) const { return p + b * sb + t * st; }
};
template <typename T> static inline View<T> view(const adn_seq& s) { return View<T>{static_cast<T*>(s.data), s.stride_b, s.stride_t}; }
template <typename T> static inline View<const T> cview(const adn_seq& s) { return View<const T>{static_cast<const T*>(s.data), s.stride_b, s.stride_t}; }

template <typename T, int V> using vec_t = T __attribute__((ext_vector_type(V)));

// vectors at any element's address: rows of an odd width start off every wider alignment, and the hardware takes that
template <typename T, int V> __device__ __forceinline__ vec_t<T, V> load_raw(const T* __restrict__ p) {
    vec_t<T, V> v;
    __builtin_memcpy(&v, p, sizeof(T) * V);
    return v;
}
template <typename T, int V> __device__ __forceinline__ void store_raw(T* __restrict__ p, const vec_t<T, V>& v) { __builtin_memcpy(p, &v, sizeof(T) * V); }
template <typename T, int V> __device__ __forceinline__ void widen(const vec_t<T, V>& v, float* out) {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = (float)v[i];
}
template <typename T, int V> __device__ __forceinline__ void load_vec(const T* __restrict__ p, float* out) {
    if constexpr (sizeof(T) * V > 16) {      // 16 bytes at a time: no wider alignment is asked for
        load_vec<T, V / 2>(p, out);
        load_vec<T, V / 2>(p + V / 2, out + V / 2);
    } else
        widen<T, V>(load_raw<T, V>(p), out);
}
// rounds to nearest even where T is bfloat16: the one rounding of a result
template <typename T, int V> __device__ __forceinline__ void store_vec(T* __restrict__ p, const float* in) {
    if constexpr (sizeof(T) * V > 16) {
        store_vec<T, V / 2>(p, in);
        store_vec<T, V / 2>(p + V / 2, in + V / 2);
        return;
    } else {
        vec_t<T, V> v;
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (T)in[i];
        store_raw<T, V>(p, v);
    }
}

// frames of utterance b that are no padding; values outside [0, T] are clamped
__device__ __forceinline__ int valid_steps(const int32_t* __restrict__ lens, int b, int T) {
    return lens ? min(max(lens[b], 0), T) : T;
}

// value of another lane: quad_perm (CTRL = p0 | p1 << 2 | p2 << 4 | p3 << 6), row_ror:n (0x120 + n) within 16 lanes, ...
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
template <int Q> __device__ __forceinline__ float quad_bcast(float v) { return dpp<Q * 0x55>(v); }
constexpr int kQuadXor1 = 0xB1, kQuadXor2 = 0x4E, kRowRor4 = 0x124, kRowRor8 = 0x128, kRowShr4 = 0x114;

// a and b, the upper 32 lanes of a exchanged with the lower 32 of b: their sum holds a's two halves added in the lower lanes, b's in
// the upper; swap16 does the same for the odd and even rows of 16 lanes
__device__ __forceinline__ float add_swap32(float a, float b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    const unsigned r0 = r[0], r1 = r[1];      // (__builtin_bit_cast of a vector's element would take element 0)
    return __builtin_bit_cast(float, r0) + __builtin_bit_cast(float, r1);
}
__device__ __forceinline__ float add_swap16(float a, float b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    const unsigned r0 = r[0], r1 = r[1];      // (__builtin_bit_cast of a vector's element would take element 0)
    return __builtin_bit_cast(float, r0) + __builtin_bit_cast(float, r1);
}
// sum over the 64 lanes, in every lane, in one fixed order
__device__ __forceinline__ float wave_sum(float v) {
    v += dpp<kQuadXor1>(v);
    v += dpp<kQuadXor2>(v);
    v += dpp<kRowRor4>(v);
    v += dpp<kRowRor8>(v);
    v = add_swap16(v, v);
    return add_swap32(v, v);
}

// 1 / (1 + exp(-x)): exact 0 and 1 at the ends (exp overflows to inf, its reciprocal is 0)
__device__ __forceinline__ float sigmoidf(float x) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * x)); }

// out segments of a sum over partial rows: segment k takes the next n columns
constexpr int kMaxSumSegs = 4;
struct SumSegs { float* out[kMaxSumSegs]; int64_t n[kMaxSumSegs]; int count; };
// out[c] = sum over p < parts of ws[p * stride + c], p in a fixed order (layernorm.hip)
int sum_parts(const float* ws, int64_t stride, int parts, const SumSegs& segs, hipStream_t s);

// a launch of `blocks` workgroups of up to 256 threads along x stays below the 2^32 threads of a dimension
static inline bool grid_ok(int64_t blocks) { return blocks < (int64_t)1 << 24; }

// dense channels, element-aligned pointer, strides that do not overlap rows are the caller's promise; this checks what can be
static inline bool seq_ok(const adn_seq& s, int elem) { return s.data && reinterpret_cast<uintptr_t>(s.data) % elem == 0; }
static inline bool seq_aligned(const adn_seq& s, int elem, int bytes) {
    return reinterpret_cast<uintptr_t>(s.data) % bytes == 0 && (s.stride_b * elem) % bytes == 0 && (s.stride_t * elem) % bytes == 0;
}
static inline bool ptr_aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace seq
}  // namespace adn
