// Root-mean-square norm with the residual's addition: forward, backward, output in 8 bits, and such rows read back.
//
//   h = x + residual,  y = h r w,  r = rsqrt(mean(h^2) + eps)
//   dx = dh + r (w dy) - h r^3 mean(h w dy),  dw = sum over rows of dy h r
//
// All of it is bound by memory: a few operations an element.  A row is held in registers between its one reading
// and its one writing: T lanes with NV vectors of 8 elements each (T = 64: a wavefront a row, no barrier; else a
// workgroup a row).  Rows of any length and address take the same path, 16-byte accesses need no alignment; only the
// vector that a row's end cuts moves element by element.  Rows beyond the registers' reach are read twice.
// dw: a workgroup takes a run of rows, its lanes keep the sums of their columns in registers; one plane of partial
// sums a workgroup, added up in the order of the planes by a second launch.  No atomics: the same bits every time.
#include "cc1d_device.hpp"
#include "cc1d_internal.hpp"
#include "cc1d_mixer.h"

namespace cc1d {
namespace {

typedef u32x4 __attribute__((aligned(2))) u32x4_any;
typedef u32x2 __attribute__((aligned(1))) u32x2_any;

template <int DT>
__device__ __forceinline__ void load8(const void *base, int64_t at, int n, float (&f)[8]) {
    using T = typename Elem<DT>::type;
    const T *x = static_cast<const T *>(base) + at;
    if (n >= 8) {
        if constexpr (DT == CC1D_F32) {
            const u32x4 a = *reinterpret_cast<const u32x4_any *>(x), b = *reinterpret_cast<const u32x4_any *>(x + 4);
            float lo[4], hi[4];
            Elem<DT>::unpack(a, lo); Elem<DT>::unpack(b, hi);
#pragma unroll
            for (int i = 0; i < 4; ++i) { f[i] = lo[i]; f[i + 4] = hi[i]; }
        } else {
            const u32x4 a = *reinterpret_cast<const u32x4_any *>(x);
            Elem<DT>::unpack(a, f);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < n ? Elem<DT>::to_float(x[i]) : 0.f;
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

__device__ __forceinline__ u32x2 pack_e4m3(const float (&f)[8]) {
    u32x2 r;
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[4], f[5], hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[6], f[7], hi, true);
    r.x = (uint32_t)lo; r.y = (uint32_t)hi;
    return r;
}

__device__ __forceinline__ float larger(float m, float a) { return a > m || a != a ? a : m; }   // a NaN stays

// The sum (or largest) of `v` over the T lanes of a row, in a fixed order.
template <int T, bool MAX>
__device__ __forceinline__ float over_row(float v, float *lds) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const float o = __shfl_xor(v, d);
        v = MAX ? larger(v, o) : v + o;
    }
    if (T == 64) return v;
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = lds[0];
#pragma unroll
    for (int i = 1; i < T / 64; ++i) r = MAX ? larger(r, lds[i]) : r + lds[i];
    __syncthreads();
    return r;
}

// XD: x and y; RD: residual and h; WD: weight; Q8: output in 8 bits.  NV = 0: a row is read twice.
template <int XD, int RD, int WD, bool Q8, int T, int NV>
__global__ void __launch_bounds__(T == 64 ? 256 : T)
norm_fwd_kernel(const cc1d_norm_params p) {
    __shared__ float lds[16];
    const int lane = threadIdx.x & (T - 1);
    const int64_t row = T == 64 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : (int64_t)blockIdx.x;
    if (T == 64 && row >= p.rows) return;
    const float over = 1.f / (float)p.dim;
    auto sum_of = [&](int c, float (&h)[8]) {            // h of the vector at column c
        const int n = p.dim - c;
        load8<XD>(p.x, row * p.x_stride + c, n, h);
        if (p.residual == nullptr) return;
        float r[8];
        load8<RD>(p.residual, row * p.residual_stride + c, n, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] += r[i];
        round8<RD>(h);
    };
    auto put = [&](int c, const float (&y)[8], float inv) {
        const int n = p.dim - c;
        if constexpr (Q8) {
            float s[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] = y[i] * inv;
            const u32x2 r = pack_e4m3(s);
            uint8_t *d = static_cast<uint8_t *>(p.y8) + row * p.y8_stride + c;
            if (n >= 8) {
                *reinterpret_cast<u32x2_any *>(d) = r;
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < n) d[i] = (uint8_t)((i < 4 ? r.x : r.y) >> (8 * (i & 3)));
            }
        } else {
            store8<XD>(p.y, row * p.y_stride + c, n, y);
        }
    };
    auto scale_of = [&](float most) {                    // writes the row's scale, returns what y is multiplied by
        if (lane == 0) p.scales[row] = most * (1.f / 448.f);
        return most > 0.f ? 448.f / most : 0.f * most;   // zeros for a row of zeros, NaN for a NaN
    };

    if constexpr (NV > 0) {
        float h[NV][8], w[NV][8], sq = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * T + lane) * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) { h[v][i] = 0.f; w[v][i] = 0.f; }
            if (c < p.dim) sum_of(c, h[v]);
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * T + lane) * 8;
            if (c < p.dim) {
                load8<WD>(p.weight, c, p.dim - c, w[v]);
                if (p.h != nullptr) store8<RD>(p.h, row * p.h_stride + c, p.dim - c, h[v]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) sq += h[v][i] * h[v][i];
        }
        const float r = rsqrtf(over_row<T, false>(sq, lds) * over + p.eps);
        float most = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                h[v][i] = h[v][i] * r * w[v][i];
                if (Q8) most = larger(most, fabsf(h[v][i]));
            }
        const float inv = Q8 ? scale_of(over_row<T, true>(most, lds)) : 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * T + lane) * 8;
            if (c < p.dim) put(c, h[v], inv);
        }
    } else {
        float sq = 0.f;
        for (int c = lane * 8; c < p.dim; c += T * 8) {
            float h[8];
            sum_of(c, h);
            if (p.h != nullptr) store8<RD>(p.h, row * p.h_stride + c, p.dim - c, h);
#pragma unroll
            for (int i = 0; i < 8; ++i) sq += h[i] * h[i];
        }
        const float r = rsqrtf(over_row<T, false>(sq, lds) * over + p.eps);
        auto value = [&](int c, float (&y)[8]) {         // each lane reads the h that it wrote
            float w[8];
            if (p.h != nullptr) load8<RD>(p.h, row * p.h_stride + c, p.dim - c, y);
            else load8<XD>(p.x, row * p.x_stride + c, p.dim - c, y);
            load8<WD>(p.weight, c, p.dim - c, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = y[i] * r * w[i];
        };
        float inv = 0.f;
        if (Q8) {
            float most = 0.f;
            for (int c = lane * 8; c < p.dim; c += T * 8) {
                float y[8];
                value(c, y);
#pragma unroll
                for (int i = 0; i < 8; ++i) most = larger(most, fabsf(y[i]));
            }
            inv = scale_of(over_row<T, true>(most, lds));
        }
        for (int c = lane * 8; c < p.dim; c += T * 8) {
            float y[8];
            value(c, y);
            put(c, y, inv);
        }
    }
}

// NV = 0: a row is read twice and dw is summed in the plane itself.
template <int XD, int RD, int WD, int T, int NV>
__global__ void __launch_bounds__(T == 64 ? 256 : T)
norm_bwd_kernel(const cc1d_norm_bwd_params p, float *planes, const int64_t rows_each) {
    __shared__ float lds[16];
    const int lane = threadIdx.x & (T - 1);
    const int64_t part = T == 64 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : (int64_t)blockIdx.x;
    const int64_t first = part * rows_each, last = first + rows_each < p.rows ? first + rows_each : p.rows;
    float *plane = planes + part * p.dim;
    const float over = 1.f / (float)p.dim;
    constexpr int N = NV > 0 ? NV : 1;
    float w[N][8], dw[N][8];
#pragma unroll
    for (int v = 0; v < N; ++v) {
        const int c = (v * T + lane) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) { w[v][i] = 0.f; dw[v][i] = 0.f; }
        if (NV > 0 && c < p.dim) load8<WD>(p.weight, c, p.dim - c, w[v]);
    }
    auto result = [&](int64_t row, int c, const float (&h)[8], const float (&wdy)[8], float r, float back) {
        const int n = p.dim - c;
        float d[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = 0.f;
        if (p.dh != nullptr) load8<RD>(p.dh, row * p.dh_stride + c, n, d);
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] += r * wdy[i] - h[i] * back;
        if (p.dx != nullptr) store8<XD>(p.dx, row * p.dx_stride + c, n, d);
        if (p.dresidual != nullptr) store8<RD>(p.dresidual, row * p.dresidual_stride + c, n, d);
    };
    for (int64_t row = first; row < last; ++row) {
        float sq = 0.f, hd = 0.f;
        if constexpr (NV > 0) {
            float h[NV][8], dy[NV][8];
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int c = (v * T + lane) * 8;
#pragma unroll
                for (int i = 0; i < 8; ++i) { h[v][i] = 0.f; dy[v][i] = 0.f; }
                if (c < p.dim) {
                    load8<RD>(p.h, row * p.h_stride + c, p.dim - c, h[v]);
                    load8<XD>(p.dy, row * p.dy_stride + c, p.dim - c, dy[v]);
                }
            }
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < 8; ++i) { sq += h[v][i] * h[v][i]; hd += h[v][i] * (w[v][i] * dy[v][i]); }
            sq = over_row<T, false>(sq, lds);
            hd = over_row<T, false>(hd, lds);
            const float r = rsqrtf(sq * over + p.eps), back = r * r * r * (hd * over);
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int c = (v * T + lane) * 8;
                float wdy[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) { dw[v][i] += dy[v][i] * (h[v][i] * r); wdy[i] = w[v][i] * dy[v][i]; }
                if (c < p.dim) result(row, c, h[v], wdy, r, back);
            }
        } else {
            for (int c = lane * 8; c < p.dim; c += T * 8) {
                float h[8], dy[8], wv[8];
                load8<RD>(p.h, row * p.h_stride + c, p.dim - c, h);
                load8<XD>(p.dy, row * p.dy_stride + c, p.dim - c, dy);
                load8<WD>(p.weight, c, p.dim - c, wv);
#pragma unroll
                for (int i = 0; i < 8; ++i) { sq += h[i] * h[i]; hd += h[i] * (wv[i] * dy[i]); }
            }
            sq = over_row<T, false>(sq, lds);
            hd = over_row<T, false>(hd, lds);
            const float r = rsqrtf(sq * over + p.eps), back = r * r * r * (hd * over);
            for (int c = lane * 8; c < p.dim; c += T * 8) {
                float h[8], dy[8], wv[8], acc[8];
                load8<RD>(p.h, row * p.h_stride + c, p.dim - c, h);
                load8<XD>(p.dy, row * p.dy_stride + c, p.dim - c, dy);
                load8<WD>(p.weight, c, p.dim - c, wv);
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[i] = 0.f;
                if (row > first) load8<CC1D_F32>(plane, c, p.dim - c, acc);
#pragma unroll
                for (int i = 0; i < 8; ++i) { acc[i] += dy[i] * (h[i] * r); wv[i] *= dy[i]; }
                store8<CC1D_F32>(plane, c, p.dim - c, acc);
                result(row, c, h, wv, r, back);
            }
        }
    }
    if constexpr (NV > 0) {
        if (first >= p.rows) return;                     // (T == 64: the last workgroup may have wavefronts without rows)
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * T + lane) * 8;
            if (c < p.dim) store8<CC1D_F32>(plane, c, p.dim - c, dw[v]);
        }
    }
}

// dweight[c] = sum of the planes, in their order: 32 columns a workgroup, 8 groups of lanes take every eighth plane.
__global__ void __launch_bounds__(256)
norm_dweight_kernel(const float *planes, const int parts, const int dim, void *dweight, const int w_dtype) {
    __shared__ float lds[8][33];
    const int col = threadIdx.x & 31, grp = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + col;
    float s = 0.f;
    if (c < dim) {
        float t[4] = {0.f, 0.f, 0.f, 0.f};
        int i = grp;
        for (; i + 24 < parts; i += 32)
#pragma unroll
            for (int j = 0; j < 4; ++j) t[j] += planes[(int64_t)(i + 8 * j) * dim + c];
        for (; i < parts; i += 8) t[0] += planes[(int64_t)i * dim + c];
        s = (t[0] + t[1]) + (t[2] + t[3]);
    }
    lds[grp][col] = s;
    __syncthreads();
    if (grp != 0 || c >= dim) return;
#pragma unroll
    for (int j = 1; j < 8; ++j) s += lds[j][col];
    if (w_dtype == CC1D_F32) static_cast<float *>(dweight)[c] = s;
    else if (w_dtype == CC1D_F16) static_cast<_Float16 *>(dweight)[c] = (_Float16)s;
    else static_cast<__bf16 *>(dweight)[c] = (__bf16)s;
}

template <int YD>
__global__ void __launch_bounds__(256)
dequantize_kernel(const cc1d_dequantize_params p, const uint32_t vecs) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row = id / vecs;
    if (row >= p.rows) return;
    const int c = (int)(id - row * vecs) * 8, n = p.dim - c;
    const uint8_t *s = static_cast<const uint8_t *>(p.y8) + row * p.y8_stride + c;
    u32x2 r;
    r.x = 0; r.y = 0;
    if (n >= 8) {
        r = *reinterpret_cast<const u32x2_any *>(s);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) { if (i < 4) r.x |= (uint32_t)s[i] << (8 * i); else r.y |= (uint32_t)s[i] << (8 * (i - 4)); }
    }
    const float scale = p.scales[row];
    float f[8];
    f[0] = __builtin_amdgcn_cvt_f32_fp8((int)r.x, 0); f[1] = __builtin_amdgcn_cvt_f32_fp8((int)r.x, 1);
    f[2] = __builtin_amdgcn_cvt_f32_fp8((int)r.x, 2); f[3] = __builtin_amdgcn_cvt_f32_fp8((int)r.x, 3);
    f[4] = __builtin_amdgcn_cvt_f32_fp8((int)r.y, 0); f[5] = __builtin_amdgcn_cvt_f32_fp8((int)r.y, 1);
    f[6] = __builtin_amdgcn_cvt_f32_fp8((int)r.y, 2); f[7] = __builtin_amdgcn_cvt_f32_fp8((int)r.y, 3);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] *= scale;
    store8<YD>(p.y, row * p.y_stride + c, n, f);
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

// Lanes of a row and vectors of 8 a lane.  A wavefront a row up to 1024 elements; then workgroups of 256, of 1024
// lanes beyond 8192 elements; beyond 16384 rows are read twice (vectors = 0).
struct RowShape { int lanes, vectors; };
RowShape row_shape(int dim) {
    if (dim <= 512) return {64, 1};
    if (dim <= 1024) return {64, 2};
    if (dim <= 2048) return {256, 1};
    if (dim <= 4096) return {256, 2};
    if (dim <= 8192) return {256, 4};
    if (dim <= 16384) return {1024, 2};
    return {1024, 0};
}
template <typename F>
int by_shape(int dim, F &&f) {
    const RowShape s = row_shape(dim);
#define CC1D_NORM_SHAPE(L, V) \
    if (s.lanes == L && s.vectors == V) return f(std::integral_constant<int, L>(), std::integral_constant<int, V>());
    CC1D_NORM_SHAPE(64, 1) CC1D_NORM_SHAPE(64, 2) CC1D_NORM_SHAPE(256, 1) CC1D_NORM_SHAPE(256, 2) CC1D_NORM_SHAPE(256, 4)
    CC1D_NORM_SHAPE(1024, 2) CC1D_NORM_SHAPE(1024, 0)
#undef CC1D_NORM_SHAPE
    return CC1D_ERR_SHAPE;
}

// Planes of partial sums: two workgroups (of 256 lanes) a CU walk the rows.
int64_t bwd_parts(int64_t rows, int dim) {
    const RowShape s = row_shape(dim);
    const int64_t most = s.lanes == 64 ? 2048 : s.lanes == 256 ? 1024 : 512;
    const int64_t each = (rows + most - 1) / most;
    return each > 0 ? (rows + each - 1) / each : 0;
}

}  // namespace
}  // namespace cc1d

using namespace cc1d;

extern "C" {

int cc1d_validate_norm(const cc1d_norm_params *p) {
    if (p == nullptr) return CC1D_ERR_NULL_POINTER;
    if (!dtype_ok(p->x_dtype) || !dtype_ok(p->r_dtype) || !dtype_ok(p->w_dtype)) return CC1D_ERR_DTYPE;
    if ((p->r_dtype != p->x_dtype && p->r_dtype != CC1D_F32) || (p->w_dtype != p->x_dtype && p->w_dtype != CC1D_F32)) return CC1D_ERR_DTYPE;
    if (p->rows < 0 || p->dim < 0) return CC1D_ERR_SHAPE;
    if (p->rows == 0 || p->dim == 0) return CC1D_OK;
    if (p->x == nullptr || p->weight == nullptr || (p->y == nullptr) == (p->y8 == nullptr)) return CC1D_ERR_NULL_POINTER;
    if ((p->residual == nullptr) != (p->h == nullptr)) return CC1D_ERR_NULL_POINTER;
    if (p->y8 != nullptr && p->scales == nullptr) return CC1D_ERR_NULL_POINTER;
    if (!on_elements(p->x, p->x_dtype) || !on_elements(p->y, p->x_dtype) || !on_elements(p->residual, p->r_dtype) ||
        !on_elements(p->h, p->r_dtype) || !on_elements(p->weight, p->w_dtype)) return CC1D_ERR_ROW_LAYOUT;
    if (p->rows >= ((int64_t)1 << 31) / 1024) return CC1D_ERR_TOO_LARGE;
    return CC1D_OK;
}

int cc1d_norm_fwd(const cc1d_norm_params *p, cc1d_stream_t stream) {
    const int st = cc1d_validate_norm(p);
    if (st != CC1D_OK || p->rows == 0 || p->dim == 0) return st;
    return by_types(p->x_dtype, p->r_dtype, p->w_dtype, [&](auto xd, auto rd, auto wd) {
        return by_shape(p->dim, [&](auto lanes, auto vectors) {
            constexpr int L = decltype(lanes)::value, V = decltype(vectors)::value;
            const dim3 grid((uint32_t)(L == 64 ? (p->rows + 3) / 4 : p->rows)), block(L == 64 ? 256 : L);
            auto go = [&](auto q8) {
                CC1D_LAUNCH((norm_fwd_kernel<decltype(xd)::value, decltype(rd)::value, decltype(wd)::value, decltype(q8)::value, L, V>),
                            grid, block, 0, static_cast<hipStream_t>(stream), *p);
                return launch_status();
            };
            return p->y8 != nullptr ? go(std::true_type()) : go(std::false_type());
        });
    });
}

int cc1d_validate_norm_bwd(const cc1d_norm_bwd_params *p) {
    if (p == nullptr) return CC1D_ERR_NULL_POINTER;
    if (!dtype_ok(p->x_dtype) || !dtype_ok(p->r_dtype) || !dtype_ok(p->w_dtype)) return CC1D_ERR_DTYPE;
    if ((p->r_dtype != p->x_dtype && p->r_dtype != CC1D_F32) || (p->w_dtype != p->x_dtype && p->w_dtype != CC1D_F32)) return CC1D_ERR_DTYPE;
    if (p->rows < 0 || p->dim < 0) return CC1D_ERR_SHAPE;
    if (p->dim == 0) return CC1D_OK;
    if (p->dweight == nullptr) return CC1D_ERR_NULL_POINTER;
    if (p->rows == 0) return CC1D_OK;
    if (p->h == nullptr || p->weight == nullptr || p->dy == nullptr) return CC1D_ERR_NULL_POINTER;
    if (!on_elements(p->h, p->r_dtype) || !on_elements(p->weight, p->w_dtype) || !on_elements(p->dy, p->x_dtype) || !on_elements(p->dh, p->r_dtype) ||
        !on_elements(p->dx, p->x_dtype) || !on_elements(p->dresidual, p->r_dtype) || !on_elements(p->dweight, p->w_dtype)) return CC1D_ERR_ROW_LAYOUT;
    return CC1D_OK;
}

int cc1d_norm_bwd_workspace_bytes(const cc1d_norm_bwd_params *p, size_t *bytes) {
    if (bytes == nullptr) return CC1D_ERR_NULL_POINTER;
    *bytes = 0;
    const int st = cc1d_validate_norm_bwd(p);
    if (st != CC1D_OK || p->dim == 0) return st;
    *bytes = (size_t)bwd_parts(p->rows, p->dim) * (size_t)p->dim * sizeof(float);
    return CC1D_OK;
}

int cc1d_norm_bwd(const cc1d_norm_bwd_params *p, void *workspace, size_t workspace_bytes, cc1d_stream_t stream) {
    size_t need = 0;
    int st = cc1d_norm_bwd_workspace_bytes(p, &need);
    if (st != CC1D_OK || p->dim == 0) return st;
    if (need > 0 && (workspace == nullptr || !aligned16(workspace) || workspace_bytes < need)) return CC1D_ERR_WORKSPACE;
    const int64_t parts = bwd_parts(p->rows, p->dim);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (p->rows > 0) {
        const int64_t each = (p->rows + parts - 1) / parts;
        st = by_types(p->x_dtype, p->r_dtype, p->w_dtype, [&](auto xd, auto rd, auto wd) {
            return by_shape(p->dim, [&](auto lanes, auto vectors) {
                constexpr int L = decltype(lanes)::value, V = decltype(vectors)::value;
                const dim3 grid((uint32_t)(L == 64 ? (parts + 3) / 4 : parts)), block(L == 64 ? 256 : L);
                CC1D_LAUNCH((norm_bwd_kernel<decltype(xd)::value, decltype(rd)::value, decltype(wd)::value, L, V>),
                            grid, block, 0, s, *p, static_cast<float *>(workspace), each);
                return launch_status();
            });
        });
        if (st != CC1D_OK) return st;
    }
    CC1D_LAUNCH(norm_dweight_kernel, dim3((uint32_t)(p->dim + 31) / 32), dim3(256), 0, s, static_cast<const float *>(workspace), (int)parts, (int)p->dim, p->dweight, (int)p->w_dtype);
    return launch_status();
}

int cc1d_validate_dequantize(const cc1d_dequantize_params *p) {
    if (p == nullptr) return CC1D_ERR_NULL_POINTER;
    if (!dtype_ok(p->y_dtype)) return CC1D_ERR_DTYPE;
    if (p->rows < 0 || p->dim < 0) return CC1D_ERR_SHAPE;
    if (p->rows == 0 || p->dim == 0) return CC1D_OK;
    if (p->y8 == nullptr || p->scales == nullptr || p->y == nullptr) return CC1D_ERR_NULL_POINTER;
    if (!on_elements(p->y, p->y_dtype)) return CC1D_ERR_ROW_LAYOUT;
    if (p->rows * ((p->dim + 7) / 8) >= ((int64_t)1 << 31)) return CC1D_ERR_TOO_LARGE;
    return CC1D_OK;
}

int cc1d_dequantize_rows(const cc1d_dequantize_params *p, cc1d_stream_t stream) {
    const int st = cc1d_validate_dequantize(p);
    if (st != CC1D_OK || p->rows == 0 || p->dim == 0) return st;
    const uint32_t vecs = (uint32_t)(p->dim + 7) / 8;
    const dim3 grid((uint32_t)((p->rows * vecs + 255) / 256));
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (p->y_dtype == CC1D_F32) CC1D_LAUNCH(dequantize_kernel<CC1D_F32>, grid, dim3(256), 0, s, *p, vecs);
    else if (p->y_dtype == CC1D_F16) CC1D_LAUNCH(dequantize_kernel<CC1D_F16>, grid, dim3(256), 0, s, *p, vecs);
    else CC1D_LAUNCH(dequantize_kernel<CC1D_BF16>, grid, dim3(256), 0, s, *p, vecs);
    return launch_status();
}

}  // extern "C"
