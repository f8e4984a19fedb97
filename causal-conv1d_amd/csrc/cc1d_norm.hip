// Root-mean-square norm with the residual's addition: forward, backward, output in 8 bits, and such rows read back.
//
//   h = x + residual,  y = h r w,  r = rsqrt(mean(h^2) + eps)
//   dx = dh + r (w dy) - h r^3 mean(h w dy),  dw = sum over rows of dy h r
//
// dx is formed as dh + r (w dy - (h r) (r mean(h w dy))), whose factors are of the size of w dy for rows of any size (r^3 is no normal
// number of 32 bits for rows of 2^42 on, and infinite below 2^-42).
// All of it is bound by memory: a few operations an element.  A row is held in registers between its one reading
// and its one writing, NV vectors of 8 elements a lane: a wavefront a row (T = 64, no barrier), else a workgroup of
// at most T lanes, as many wavefronts as the row fills.  Rows of any length and address take the same path, 16-byte
// accesses need no alignment; only the vector that a row's end cuts moves element by element.  Rows beyond the
// registers' reach are read twice.  The barriers between a row's wavefronts order LDS alone, so that h is still on its
// way to memory while the row is summed.
// dw: a workgroup takes a run of rows, its lanes keep the sums of their columns in registers; one plane of partial sums a
// workgroup, added up in the order of the planes by a second launch.  No atomics: the same bits every time.
//
// 16384 rows of 2560, residual in fp32: forward 99 to 106 us (4.7 to 5.1 TB/s), backward 122 (5.5) and 4.7 for dw's planes.  To 8 bits, 8192 rows of
// 5120: 48 us (6.1 TB/s), and 20 back.  64 such rows: 4.7 us and 2.6, a launch, two reductions and a barrier each.
#include "cc1d_rows.hpp"

namespace cc1d {
namespace {

typedef u32x2 __attribute__((aligned(1))) u32x2_any;

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

// a / b to nearest, with inv = 1 / b to nearest: a product that is off by two units in the last place at most, and its rest, which is exact.
// (4e8 random pairs, mantissas of b near 1 and 2 among them, against the division: equal.)  A product with inv alone is off in every fourth
// pair, and a code of 8 bits is then the wrong one next to a tie.  Three instructions more, hidden behind memory.
__device__ __forceinline__ float quotient(float a, float b, float inv) {
    const float q = a * inv;
    return fmaf(-fmaf(q, b, -a), inv, q);                // (in these signs a zero keeps its own)
}

// XD: x and y; RD: residual and h; WD: weight; Q8: output in 8 bits.  NV = 0: a row is read twice.
template <int XD, int RD, int WD, bool Q8, int T, int NV>
__global__ void __launch_bounds__(threads_of(T))
norm_fwd_kernel(const cc1d_norm_params p, const int64_t first, const int64_t last) {
    __shared__ float lds[2][16];
    const int lane = T == 64 ? (int)(threadIdx.x & 63) : (int)threadIdx.x, lanes = T == 64 ? 64 : (int)blockDim.x;
    const int64_t row = first + (T == 64 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : (int64_t)blockIdx.x);
    if (T == 64 && row >= last) return;
    const float over = 1.f / (float)p.dim;
    float up = 1.f, by = 1.f, inv = 1.f;                 // in 8 bits: y up / by, and 1 / by
    auto put = [&](int c, const float (&y)[8]) {
        const int n = p.dim - c;
        if constexpr (Q8) {
            float s[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] = quotient(y[i] * up, by, inv);
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
    // Writes the row's scale, and what y is divided by: the scale as it is stored, so that a code is the one next to y / scale.  Where that is
    // so small that a quotient's rest or the scale itself would be no normal number, both are 2^96 times as large (the scale
    // before it is rounded to one of those that are not).  A row of zeros is divided by 1; over an infinity all that is finite is 0.
    auto scale_of = [&](float most) {
        if (most < 0x1p-64f) up = 0x1p96f;
        if (lane == 0) p.scales[row] = most * (1.f / 448.f);
        by = most == 0.f ? 1.f : most * up * (1.f / 448.f);
        inv = 1.f / by;
        if (inv == 0.f) by = 0.f;
    };

    if constexpr (NV > 0) {
        Raw8<XD, Q8> x[NV];
        Raw8<RD, Q8> res[NV];
        Raw8<WD> w[NV];
        float h[NV][8], sq = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) x[v].load(p.x, row * p.x_stride, (v * lanes + lane) * 8, p.dim);
        if (p.residual != nullptr) {
#pragma unroll
            for (int v = 0; v < NV; ++v) res[v].load(p.residual, row * p.residual_stride, (v * lanes + lane) * 8, p.dim);
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) w[v].load(p.weight, 0, (v * lanes + lane) * 8, p.dim);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * lanes + lane) * 8;
            x[v].to(h[v]);
            if (p.residual != nullptr) {
                float r[8];
                res[v].to(r);
#pragma unroll
                for (int i = 0; i < 8; ++i) h[v][i] += r[i];
                round8<RD>(h[v]);
                if (c < p.dim) store8<RD>(p.h, row * p.h_stride + c, p.dim - c, h[v]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) sq += h[v][i] * h[v][i];
        }
        const float r = rsqrtf(over_row<T, false>(sq, lds[0]) * over + p.eps);
        float most = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            float wf[8];
            w[v].to(wf);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                h[v][i] = h[v][i] * r * wf[i];
                if (Q8) most = larger(most, fabsf(h[v][i]));
            }
        }
        if (Q8) scale_of(over_row<T, true>(most, lds[1]));
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * lanes + lane) * 8;
            if (c < p.dim) put(c, h[v]);
        }
    } else {
        float sq = 0.f;
        for (int c = lane * 8; c < p.dim; c += lanes * 8) {
            float h[8];
            load8<XD>(p.x, row * p.x_stride, c, p.dim, h);
            if (p.residual != nullptr) {
                float r[8];
                load8<RD>(p.residual, row * p.residual_stride, c, p.dim, r);
#pragma unroll
                for (int i = 0; i < 8; ++i) h[i] += r[i];
                round8<RD>(h);
                store8<RD>(p.h, row * p.h_stride + c, p.dim - c, h);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) sq += h[i] * h[i];
        }
        const float r = rsqrtf(over_row<T, false>(sq, lds[0]) * over + p.eps);
        auto value = [&](int c, float (&y)[8]) {         // each lane reads the h that it wrote
            float w[8];
            if (p.h != nullptr) load8<RD>(p.h, row * p.h_stride, c, p.dim, y);
            else load8<XD>(p.x, row * p.x_stride, c, p.dim, y);
            load8<WD>(p.weight, 0, c, p.dim, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = y[i] * r * w[i];
        };
        if (Q8) {
            float most = 0.f;
            for (int c = lane * 8; c < p.dim; c += lanes * 8) {
                float y[8];
                value(c, y);
#pragma unroll
                for (int i = 0; i < 8; ++i) most = larger(most, fabsf(y[i]));
            }
            scale_of(over_row<T, true>(most, lds[1]));
        }
        for (int c = lane * 8; c < p.dim; c += lanes * 8) {
            float y[8];
            value(c, y);
            put(c, y);
        }
    }
}

// A workgroup takes rows_each rows, its wavefronts every fourth of them where a wavefront takes a row.
// NV = 0: a row is read twice and dw is summed in the plane itself.
template <int XD, int RD, int WD, int T, int NV>
__global__ void __launch_bounds__(threads_of(T))
norm_bwd_kernel(const cc1d_norm_bwd_params p, float *planes, const int64_t rows_each) {
    __shared__ float lds[2][2][16];
    const int lane = T == 64 ? (int)(threadIdx.x & 63) : (int)threadIdx.x, lanes = T == 64 ? 64 : (int)blockDim.x;
    const int wave = threadIdx.x >> 6;
    const int64_t begin = blockIdx.x * rows_each, last = begin + rows_each < p.rows ? begin + rows_each : p.rows;
    const int64_t first = begin + (T == 64 ? wave : 0);
    constexpr int step = T == 64 ? 4 : 1;
    float *plane = planes + (int64_t)blockIdx.x * p.dim;
    const float over = 1.f / (float)p.dim;
    auto put = [&](int64_t row, int c, const float (&d)[8]) {
        const int n = p.dim - c;
        if (p.dx != nullptr) store8<XD>(p.dx, row * p.dx_stride + c, n, d);
        if (p.dresidual != nullptr) store8<RD>(p.dresidual, row * p.dresidual_stride + c, n, d);
    };
    int turn = 0;                                        // which half of `lds`: a row's sums may still be read when the next one's are written
    auto over_rows_waves = [&](float &sq, float &hd) {
        sq = over_lanes<false>(sq);
        hd = over_lanes<false>(hd);
        if constexpr (T > 64) {
            const int waves = blockDim.x >> 6;
            if ((threadIdx.x & 63) == 0) { lds[turn][0][wave] = sq; lds[turn][1][wave] = hd; }
            lds_barrier();
            sq = lds[turn][0][0];
            hd = lds[turn][1][0];
            for (int i = 1; i < waves; ++i) { sq += lds[turn][0][i]; hd += lds[turn][1][i]; }
            turn ^= 1;
        }
    };
    if constexpr (NV > 0) {
        Raw8<WD> wr[NV];
        Raw8<RD, true> hr[NV], dhr[NV];
        Raw8<XD, true> dyr[NV];
        auto ask = [&](int64_t row) {
#pragma unroll
            for (int v = 0; v < NV; ++v) hr[v].load(p.h, row * p.h_stride, (v * lanes + lane) * 8, p.dim);
#pragma unroll
            for (int v = 0; v < NV; ++v) dyr[v].load(p.dy, row * p.dy_stride, (v * lanes + lane) * 8, p.dim);
            if (p.dh != nullptr) {
#pragma unroll
                for (int v = 0; v < NV; ++v) dhr[v].load(p.dh, row * p.dh_stride, (v * lanes + lane) * 8, p.dim);
            }
        };
        float w[NV][8], dw[NV][8];
#pragma unroll
        for (int v = 0; v < NV; ++v) wr[v].load(p.weight, 0, (v * lanes + lane) * 8, p.dim);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            wr[v].to(w[v]);
#pragma unroll
            for (int i = 0; i < 8; ++i) dw[v][i] = 0.f;
        }
        for (int64_t row = first; row < last; row += step) {
            float h[NV][8], dy[NV][8], d[NV][8], sq = 0.f, hd = 0.f;
            ask(row);
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                hr[v].to(h[v]);
                dyr[v].to(dy[v]);
#pragma unroll
                for (int i = 0; i < 8; ++i) d[v][i] = 0.f;
                if (p.dh != nullptr) dhr[v].to(d[v]);
            }
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < 8; ++i) { sq += h[v][i] * h[v][i]; hd += h[v][i] * (w[v][i] * dy[v][i]); }
            over_rows_waves(sq, hd);
            const float r = rsqrtf(sq * over + p.eps), back = hd * over * r;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int c = (v * lanes + lane) * 8;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float unit = h[v][i] * r;
                    dw[v][i] += dy[v][i] * unit;
                    d[v][i] += r * (w[v][i] * dy[v][i] - unit * back);
                }
                if (c < p.dim) put(row, c, d[v]);
            }
        }
        if constexpr (T == 64) {                         // the four wavefronts' sums, in their order
            __shared__ float sums[4][NV * 64 * 8];
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < 8; ++i) sums[wave][(v * 8 + i) * 64 + lane] = dw[v][i];
            lds_barrier();
            for (int k = threadIdx.x; k < NV * 64 * 8; k += 256) {
                const int c = ((k >> 9) * 64 + (k & 63)) * 8 + ((k >> 6) & 7);
                if (c < p.dim) plane[c] = (sums[0][k] + sums[1][k]) + (sums[2][k] + sums[3][k]);
            }
        } else {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int c = (v * lanes + lane) * 8;
                if (c < p.dim) store8<CC1D_F32>(plane, c, p.dim - c, dw[v]);
            }
        }
    } else {
        for (int64_t row = first; row < last; row += step) {
            float sq = 0.f, hd = 0.f;
            for (int c = lane * 8; c < p.dim; c += lanes * 8) {
                float h[8], dy[8], wv[8];
                load8<RD>(p.h, row * p.h_stride, c, p.dim, h);
                load8<XD>(p.dy, row * p.dy_stride, c, p.dim, dy);
                load8<WD>(p.weight, 0, c, p.dim, wv);
#pragma unroll
                for (int i = 0; i < 8; ++i) { sq += h[i] * h[i]; hd += h[i] * (wv[i] * dy[i]); }
            }
            over_rows_waves(sq, hd);
            const float r = rsqrtf(sq * over + p.eps), back = hd * over * r;
            for (int c = lane * 8; c < p.dim; c += lanes * 8) {
                float h[8], dy[8], wv[8], acc[8], d[8];
                load8<RD>(p.h, row * p.h_stride, c, p.dim, h);
                load8<XD>(p.dy, row * p.dy_stride, c, p.dim, dy);
                load8<WD>(p.weight, 0, c, p.dim, wv);
#pragma unroll
                for (int i = 0; i < 8; ++i) { acc[i] = 0.f; d[i] = 0.f; }
                if (row > first) load8<CC1D_F32>(plane, 0, c, p.dim, acc);
                if (p.dh != nullptr) load8<RD>(p.dh, row * p.dh_stride, c, p.dim, d);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float unit = h[i] * r;
                    acc[i] += dy[i] * unit;
                    d[i] += r * (wv[i] * dy[i] - unit * back);
                }
                store8<CC1D_F32>(plane, c, p.dim - c, acc);
                put(row, c, d);
            }
        }
    }
}

template <int YD>
__global__ void __launch_bounds__(256)
dequantize_kernel(const cc1d_dequantize_params p, const uint32_t vecs, const int64_t first, const int64_t last) {
    const uint32_t id = blockIdx.x * 256u + threadIdx.x;
    const int64_t row = first + id / vecs;
    if (row >= last) return;
    const int c = (int)(id % vecs) * 8, n = p.dim - c;
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

// Workgroups of the backward on a CU: 1024 lanes (16384 rows of 2560: three
// of 320 lanes 122 us, two 127, four 151: too many rows at once).
int bwd_a_cu(int dim) { return 1024 / bwd_lanes(dim); }

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
    if (p->dim > kLongestRow) return CC1D_ERR_TOO_LARGE;
    if (p->x == nullptr || p->weight == nullptr || (p->y == nullptr) == (p->y8 == nullptr)) return CC1D_ERR_NULL_POINTER;
    if ((p->residual == nullptr) != (p->h == nullptr)) return CC1D_ERR_NULL_POINTER;
    if (p->y8 != nullptr && p->scales == nullptr) return CC1D_ERR_NULL_POINTER;
    if (!on_elements(p->x, p->x_dtype) || !on_elements(p->y, p->x_dtype) || !on_elements(p->residual, p->r_dtype) ||
        !on_elements(p->h, p->r_dtype) || !on_elements(p->weight, p->w_dtype)) return CC1D_ERR_ROW_LAYOUT;
    return CC1D_OK;
}

int cc1d_norm_fwd(const cc1d_norm_params *p, cc1d_stream_t stream) {
    const int st = cc1d_validate_norm(p);
    if (st != CC1D_OK || p->rows == 0 || p->dim == 0) return st;
    return by_types(p->x_dtype, p->r_dtype, p->w_dtype, [&](auto xd, auto rd, auto wd) {
        return by_shape(fwd_shape(p->dim), [&](auto lanes, auto vectors) {
            constexpr int L = decltype(lanes)::value, V = decltype(vectors)::value;
            const int lanes_of_block = L == 64 ? 256 : fwd_shape(p->dim).lanes, rows_of_block = L == 64 ? 4 : 1;
            const int64_t blocks = thread_limit() / lanes_of_block, slice = (blocks > 1 ? blocks : 1) * rows_of_block;
            auto go = [&](auto q8) {
                for (int64_t first = 0; first < p->rows; first += slice) {
                    const int64_t last = p->rows - first > slice ? first + slice : p->rows;
                    CC1D_LAUNCH((norm_fwd_kernel<decltype(xd)::value, decltype(rd)::value, decltype(wd)::value, decltype(q8)::value, L, V>),
                                dim3((uint32_t)((last - first + rows_of_block - 1) / rows_of_block)), dim3(lanes_of_block), 0,
                                static_cast<hipStream_t>(stream), *p, first, last);
                    const int st = launch_status();
                    if (st != CC1D_OK) return st;
                }
                return (int)CC1D_OK;
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
    if (p->dim > kLongestRowBwd) return CC1D_ERR_TOO_LARGE;
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
    *bytes = (size_t)bwd_parts(p->rows, bwd_a_cu(p->dim)) * (size_t)p->dim * sizeof(float);
    return CC1D_OK;
}

int cc1d_norm_bwd(const cc1d_norm_bwd_params *p, void *workspace, size_t workspace_bytes, cc1d_stream_t stream) {
    size_t need = 0;
    int st = cc1d_norm_bwd_workspace_bytes(p, &need);
    if (st != CC1D_OK || p->dim == 0) return st;
    if (need > 0 && (workspace == nullptr || !aligned16(workspace) || workspace_bytes < need)) return CC1D_ERR_WORKSPACE;
    const int64_t parts = bwd_parts(p->rows, bwd_a_cu(p->dim));
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (p->rows > 0) {
        const int64_t each = (p->rows + parts - 1) / parts;
        st = by_types(p->x_dtype, p->r_dtype, p->w_dtype, [&](auto xd, auto rd, auto wd) {
            return by_shape(bwd_shape(p->dim), [&](auto lanes, auto vectors) {
                constexpr int L = decltype(lanes)::value, V = decltype(vectors)::value;
                CC1D_LAUNCH((norm_bwd_kernel<decltype(xd)::value, decltype(rd)::value, decltype(wd)::value, L, V>),
                            dim3((uint32_t)parts), dim3(L == 64 ? 256 : bwd_shape(p->dim).lanes), 0, s, *p, static_cast<float *>(workspace), each);
                return launch_status();
            });
        });
        if (st != CC1D_OK) return st;
    }
    CC1D_LAUNCH(norm_dweight_kernel, dim3((uint32_t)(p->dim + 31) / 32), dim3(1024), 0, s, static_cast<const float *>(workspace), (int)parts, (int)p->dim, (int)p->dim,
                p->dweight, (void *)nullptr, (int)p->w_dtype);
    return launch_status();
}

int cc1d_validate_dequantize(const cc1d_dequantize_params *p) {
    if (p == nullptr) return CC1D_ERR_NULL_POINTER;
    if (!dtype_ok(p->y_dtype)) return CC1D_ERR_DTYPE;
    if (p->rows < 0 || p->dim < 0) return CC1D_ERR_SHAPE;
    if (p->rows == 0 || p->dim == 0) return CC1D_OK;
    if (p->y8 == nullptr || p->scales == nullptr || p->y == nullptr) return CC1D_ERR_NULL_POINTER;
    if (!on_elements(p->y, p->y_dtype)) return CC1D_ERR_ROW_LAYOUT;
    return CC1D_OK;
}

int cc1d_dequantize_rows(const cc1d_dequantize_params *p, cc1d_stream_t stream) {
    const int st = cc1d_validate_dequantize(p);
    if (st != CC1D_OK || p->rows == 0 || p->dim == 0) return st;
    const uint32_t vecs = ((uint32_t)p->dim + 7) / 8;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t slice = thread_limit() / vecs > 1 ? thread_limit() / vecs : 1;         // (a row has at most 2^28 vectors)
    for (int64_t first = 0; first < p->rows; first += slice) {
        const int64_t last = p->rows - first > slice ? first + slice : p->rows;
        const dim3 grid((uint32_t)(((last - first) * vecs + 255) / 256));
        if (p->y_dtype == CC1D_F32) CC1D_LAUNCH(dequantize_kernel<CC1D_F32>, grid, dim3(256), 0, s, *p, vecs, first, last);
        else if (p->y_dtype == CC1D_F16) CC1D_LAUNCH(dequantize_kernel<CC1D_F16>, grid, dim3(256), 0, s, *p, vecs, first, last);
        else CC1D_LAUNCH(dequantize_kernel<CC1D_BF16>, grid, dim3(256), 0, s, *p, vecs, first, last);
        const int st = launch_status();
        if (st != CC1D_OK) return st;
    }
    return CC1D_OK;
}

}  // extern "C"
