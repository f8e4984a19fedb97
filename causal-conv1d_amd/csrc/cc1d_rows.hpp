// What the norms' kernels share: rows of any length, type and address in registers, sums over a row, the shapes of workgroups, and the sum of
// partial sums over planes.
#pragma once

#include "cc1d_device.hpp"
#include "cc1d_internal.hpp"
#include "cc1d_mixer.h"

#include <type_traits>

namespace cc1d {
namespace {

typedef u32x4 __attribute__((aligned(2))) u32x4_any;

// Eight elements of a row of `dim`, from column c, as they lie in memory; zeros behind the row's end.  The load that
// every lane makes has no condition (lanes without a vector of their own repeat the row's first), so loads that follow
// each other travel together.  LAST: nobody reads these bytes after this kernel, the caches
// need not keep them.  The backward of 16384 rows of 2560 takes 122 us with it and 140 without, the output in 8 bits of 8192
// rows of 5120 49 and 54; the plain forward, 99 and 93, goes without.
template <int DT, bool LAST = false>
struct Raw8 {
    using T = typename Elem<DT>::type;
    T x[8];
    __device__ __forceinline__ static u32x4 read(const T *p) {
        const u32x4_any *q = reinterpret_cast<const u32x4_any *>(p);
        return LAST ? __builtin_nontemporal_load(q) : *q;
    }
    __device__ __forceinline__ void load(const void *base, int64_t row, int c, int dim) {
        const T *r = static_cast<const T *>(base) + row;
        const int n = dim - c;
        if (dim >= 8) {
            const T *from = r + (n >= 8 ? c : 0);
            u32x4 *to = reinterpret_cast<u32x4 *>(x);
            to[0] = read(from);
            if constexpr (DT == CC1D_F32) to[1] = read(from + 4);
        }
        if (n < 8) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = T(0);
            if (n > 0) {
#pragma unroll
                for (int i = 0; i < 7; ++i)
                    if (i < n) x[i] = r[c + i];
            }
        }
    }
    __device__ __forceinline__ void to(float (&f)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = Elem<DT>::to_float(x[i]);
    }
};
template <int DT>
__device__ __forceinline__ void load8(const void *base, int64_t row, int c, int dim, float (&f)[8]) {
    Raw8<DT> r;
    r.load(base, row, c, dim);
    r.to(f);
}

template <int DT>
__device__ __forceinline__ void store8(void *base, int64_t at, int n, const float (&f)[8]) {
    using T = typename Elem<DT>::type;
    T *x = static_cast<T *>(base) + at;
    if (n >= 8) {
        if constexpr (DT == CC1D_F32) {
            float lo[4], hi[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) { lo[i] = f[i]; hi[i] = f[i + 4]; }
            *reinterpret_cast<u32x4_any *>(x) = Elem<DT>::pack(lo);
            *reinterpret_cast<u32x4_any *>(x + 4) = Elem<DT>::pack(hi);
        } else {
            *reinterpret_cast<u32x4_any *>(x) = Elem<DT>::pack(f);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) x[i] = Elem<DT>::from_float(f[i]);
}

// What f becomes in type DT.
template <int DT>
__device__ __forceinline__ void round8(float (&f)[8]) {
    if constexpr (DT != CC1D_F32) {
        const u32x4 r = Elem<DT>::pack(f);
        Elem<DT>::unpack(r, f);
    }
}

__device__ __forceinline__ float larger(float m, float a) { return a > m || a != a ? a : m; }   // a NaN stays

template <bool MAX>
__device__ __forceinline__ float joined(float a, float b) { return MAX ? larger(a, b) : a + b; }
// The sum (or largest) over a wavefront, by DPP and half swaps, in a fixed order.
template <bool MAX>
__device__ __forceinline__ float over_lanes(float v) {
    v = joined<MAX>(v, dpp_moved<0xB1>(v));              // quad_perm: lane ^ 1
    v = joined<MAX>(v, dpp_moved<0x4E>(v));              // lane ^ 2
    v = joined<MAX>(v, dpp_moved<0x124>(v));             // row_ror:4
    v = joined<MAX>(v, dpp_moved<0x128>(v));             // row_ror:8
    const auto a = __builtin_amdgcn_permlane16_swap(bitcast<uint32_t>(v), bitcast<uint32_t>(v), false, false);
    v = joined<MAX>(bitcast<float>((uint32_t)a[0]), bitcast<float>((uint32_t)a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(bitcast<uint32_t>(v), bitcast<uint32_t>(v), false, false);
    return joined<MAX>(bitcast<float>((uint32_t)b[0]), bitcast<float>((uint32_t)b[1]));
}
// The same over a row's wavefronts; `lds` is for this sum alone.
template <int T, bool MAX>
__device__ __forceinline__ float over_row(float v, float *lds) {
    v = over_lanes<MAX>(v);
    if constexpr (T > 64) {
        const int waves = blockDim.x >> 6;
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        lds_barrier();
        v = lds[0];
        for (int i = 1; i < waves; ++i) v = joined<MAX>(v, lds[i]);
    }
    return v;
}

// Sums of several numbers at once, one barrier, the same bits in every lane (the lanes' own orders of over_lanes may part them by a rounding); `lds` is for
// these alone.
template <int T, int N>
__device__ __forceinline__ void over_row(float (&v)[N], float (*lds)[16]) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = bitcast<float>(__builtin_amdgcn_readfirstlane(bitcast<int>(over_lanes<false>(v[k]))));
    if constexpr (T > 64) {
        const int waves = blockDim.x >> 6;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int k = 0; k < N; ++k) lds[k][threadIdx.x >> 6] = v[k];
        }
        lds_barrier();
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = lds[k][0];
        for (int i = 1; i < waves; ++i) {
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] += lds[k][i];
        }
    }
}

constexpr int threads_of(int T) { return T == 64 ? 256 : T; }

// The sum of the planes of `width` columns, in a fixed order: 32 columns a workgroup, 32 groups of lanes take every 32nd plane, 8 at a time.  The
// first dim columns are dweight, those behind them dbias.
__global__ void __launch_bounds__(1024)
norm_dweight_kernel(const float *planes, const int parts, const int width, const int dim, void *dweight, void *dbias, const int w_dtype) {
    __shared__ float lds[32][33];
    const int col = threadIdx.x & 31, grp = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + col;
    float t[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (c < width) {
        for (int i = grp; i < parts; i += 256) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = planes[(int64_t)(i + 32 * j < parts ? i + 32 * j : i) * width + c];
#pragma unroll
            for (int j = 0; j < 8; ++j) t[j] += i + 32 * j < parts ? x[j] : 0.f;
        }
    }
    lds[grp][col] = ((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7]));
    __syncthreads();
    if (grp != 0 || c >= width) return;
    float s = lds[0][col];
#pragma unroll
    for (int j = 1; j < 32; ++j) s += lds[j][col];
    void *to = c < dim ? dweight : dbias;
    const int at = c < dim ? c : c - dim;
    if (w_dtype == CC1D_F32) static_cast<float *>(to)[at] = s;
    else if (w_dtype == CC1D_F16) static_cast<_Float16 *>(to)[at] = (_Float16)s;
    else static_cast<__bf16 *>(to)[at] = (__bf16)s;
}

bool dtype_ok(int d) { return d == CC1D_F32 || d == CC1D_F16 || d == CC1D_BF16; }
bool on_elements(const void *p, int dtype) { return (reinterpret_cast<uintptr_t>(p) & ((uintptr_t)elem_bytes(dtype) - 1)) == 0; }

// The types that meet in practice: residual and weight each in x's type or in fp32.
template <typename F>
int by_types(int xd, int rd, int wd, F &&f) {
    if ((rd != xd && rd != CC1D_F32) || (wd != xd && wd != CC1D_F32)) return CC1D_ERR_DTYPE;
#define CC1D_NORM_TYPES(X)                                                                                              \
    if (xd == X) {                                                                                                      \
        if (rd == X && wd == X) return f(std::integral_constant<int, X>(), std::integral_constant<int, X>(), std::integral_constant<int, X>()); \
        if (rd == X) return f(std::integral_constant<int, X>(), std::integral_constant<int, X>(), std::integral_constant<int, CC1D_F32>());     \
        if (wd == X) return f(std::integral_constant<int, X>(), std::integral_constant<int, CC1D_F32>(), std::integral_constant<int, X>());     \
        return f(std::integral_constant<int, X>(), std::integral_constant<int, CC1D_F32>(), std::integral_constant<int, CC1D_F32>());           \
    }
    if (xd == CC1D_F32) return f(std::integral_constant<int, CC1D_F32>(), std::integral_constant<int, CC1D_F32>(), std::integral_constant<int, CC1D_F32>());
    CC1D_NORM_TYPES(CC1D_F16)
    CC1D_NORM_TYPES(CC1D_BF16)
#undef CC1D_NORM_TYPES
    return CC1D_ERR_DTYPE;
}

// How a row lies in registers.  A wavefront a row up to 1024 elements; then a workgroup of as many wavefronts as the
// row takes at `vectors` a lane; beyond 16384 elements rows are read twice (vectors = 0).
struct RowShape { int most_lanes, vectors, lanes; };
RowShape row_shape(int dim, int vectors) {
    if (dim <= 512) return {64, 1, 64};
    if (dim <= 1024) return {64, 2, 64};
    if (dim > 16384) return {1024, 0, 1024};
    if (dim > 8192) vectors = 2;
    const int lanes = (dim + 512 * vectors - 1) / (512 * vectors) * 64;
    return {lanes <= 512 ? 512 : 1024, vectors, lanes};
}
// Lanes step along such a row by 1024 vectors, and a step has to stay within 32 bits; norm_dweight_kernel takes 1024 threads for 32 columns, and a
// launch has fewer than 2^32.
constexpr int kLongestRow = INT32_MAX - 1024 * 8, kLongestRowBwd = (1 << 27) - 32;
RowShape fwd_shape(int dim) { return row_shape(dim, 2); }
RowShape bwd_shape(int dim) { return row_shape(dim, 1); }
template <typename F>
int by_shape(const RowShape &s, F &&f) {
#define CC1D_NORM_SHAPE(L, V) \
    if (s.most_lanes == L && s.vectors == V) return f(std::integral_constant<int, L>(), std::integral_constant<int, V>());
    CC1D_NORM_SHAPE(64, 1) CC1D_NORM_SHAPE(64, 2) CC1D_NORM_SHAPE(512, 1) CC1D_NORM_SHAPE(512, 2) CC1D_NORM_SHAPE(1024, 1)
    CC1D_NORM_SHAPE(1024, 2) CC1D_NORM_SHAPE(1024, 0)
#undef CC1D_NORM_SHAPE
    return CC1D_ERR_SHAPE;
}

// Planes of partial sums, one a workgroup: `a_cu` workgroups a CU, and no fewer than four rows to each.
int bwd_lanes(int dim) { const int lanes = bwd_shape(dim).lanes; return lanes == 64 ? 256 : lanes; }
int64_t bwd_parts(int64_t rows, int a_cu) {
    const int64_t most = 256 * (a_cu > 1 ? a_cu : 1);
    int64_t each = (rows + most - 1) / most;
    if (each < 4) each = 4;
    return (rows + each - 1) / each;
}

}  // namespace
}  // namespace cc1d
