// Layer norm with the residual's addition: forward and backward.
//
//   h = x + residual,  n = (h - mean(h)) r,  r = rsqrt(mean((h - mean(h))^2) + eps),  y = n w + b
//   dx = dh + r (w dy - mean(w dy) - n mean(w dy n)),  dw = sum over rows of dy n,  db = sum over rows of dy
//
// Rows lie in registers as the root-mean-square norm's do (cc1d_norm.hip), and memory bounds it as well.  The mean goes first and the squares are those of
// differences, two sums one behind the other: of a row whose mean is large beside its spread, mean(h^2) - mean(h)^2 would leave nothing.  The mean itself is
// rounded, by up to some 2^-22 of it, which may be more than the spread: the differences' own mean, one more sum beside that of their squares, is taken off
// them (2560 numbers of 100003, whose y is the bias: off by 0.43 without).  A training forward leaves each row's mean and r for the backward, 8 bytes a row, which saves that one its first pair of
// sums; the differences' mean it makes anew beside its own two.
// db's partial sums lie behind dw's in the same planes.
//
// 16384 rows of 2560, residual in fp32: forward 118 us (4.3 TB/s; 107 at best), backward 134 (5.0; 128) and 5 for the planes; 8192 of 5120, bfloat16: 62 (5.4); 64 such rows: 4.6 us, a
// launch and two reductions one behind the other.
#include "cc1d_rows.hpp"

namespace cc1d {
namespace {

// The difference of two sums may come out below 0; a NaN stays.
__device__ __forceinline__ float reciprocal_spread(float variance, float eps) { return rsqrtf((variance < 0.f ? 0.f : variance) + eps); }

// XD: x and y; RD: residual and h; WD: weight and bias.  NV = 0: a row is read three times.
template <int XD, int RD, int WD, int T, int NV>
__global__ void __launch_bounds__(threads_of(T))
layer_norm_fwd_kernel(const cc1d_layer_norm_params p, const int64_t first, const int64_t last) {
    __shared__ float lds[3][16];
    const int lane = T == 64 ? (int)(threadIdx.x & 63) : (int)threadIdx.x, lanes = T == 64 ? 64 : (int)blockDim.x;
    const int64_t row = first + (T == 64 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : (int64_t)blockIdx.x);
    if (T == 64 && row >= last) return;
    const float over = 1.f / (float)p.dim;
    auto keep = [&](float mean, float r) {
        if (p.stats != nullptr && lane == 0) *reinterpret_cast<float2 *>(p.stats + 2 * row) = make_float2(mean, r);
    };

    if constexpr (NV > 0) {
        Raw8<XD> x[NV];
        Raw8<RD> res[NV];
        Raw8<WD> w[NV], b[NV];
        float h[NV][8], sum[1] = {0.f}, of_differences[2] = {0.f, 0.f};  // their sum, and of their squares
#pragma unroll
        for (int v = 0; v < NV; ++v) x[v].load(p.x, row * p.x_stride, (v * lanes + lane) * 8, p.dim);
        if (p.residual != nullptr) {
#pragma unroll
            for (int v = 0; v < NV; ++v) res[v].load(p.residual, row * p.residual_stride, (v * lanes + lane) * 8, p.dim);
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) w[v].load(p.weight, 0, (v * lanes + lane) * 8, p.dim);
        if (p.bias != nullptr) {
#pragma unroll
            for (int v = 0; v < NV; ++v) b[v].load(p.bias, 0, (v * lanes + lane) * 8, p.dim);
        }
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
            for (int i = 0; i < 8; ++i) sum[0] += h[v][i];
        }
        over_row<T>(sum, lds);
        const float mean = sum[0] * over;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int n = p.dim - (v * lanes + lane) * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                h[v][i] = i < n ? h[v][i] - mean : 0.f;
                of_differences[0] += h[v][i];
                of_differences[1] += h[v][i] * h[v][i];
            }
        }
        over_row<T>(of_differences, lds + 1);
        const float off = of_differences[0] * over, r = reciprocal_spread(of_differences[1] * over - off * off, p.eps);
        keep(mean, r);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * lanes + lane) * 8;
            float wf[8], bf[8];
            w[v].to(wf);
#pragma unroll
            for (int i = 0; i < 8; ++i) bf[i] = 0.f;
            if (p.bias != nullptr) b[v].to(bf);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[v][i] = fmaf((h[v][i] - off) * r, wf[i], bf[i]);
            if (c < p.dim) store8<XD>(p.y, row * p.y_stride + c, p.dim - c, h[v]);
        }
    } else {
        float sum[1] = {0.f}, of_differences[2] = {0.f, 0.f};
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
            for (int i = 0; i < 8; ++i) sum[0] += h[i];
        }
        over_row<T>(sum, lds);
        const float mean = sum[0] * over;
        auto centred = [&](int c, float (&h)[8]) {       // each lane reads the h that it wrote
            if (p.h != nullptr) load8<RD>(p.h, row * p.h_stride, c, p.dim, h);
            else load8<XD>(p.x, row * p.x_stride, c, p.dim, h);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = i < p.dim - c ? h[i] - mean : 0.f;
        };
        for (int c = lane * 8; c < p.dim; c += lanes * 8) {
            float h[8];
            centred(c, h);
#pragma unroll
            for (int i = 0; i < 8; ++i) { of_differences[0] += h[i]; of_differences[1] += h[i] * h[i]; }
        }
        over_row<T>(of_differences, lds + 1);
        const float off = of_differences[0] * over, r = reciprocal_spread(of_differences[1] * over - off * off, p.eps);
        keep(mean, r);
        for (int c = lane * 8; c < p.dim; c += lanes * 8) {
            float h[8], w[8], b[8];
            centred(c, h);
            load8<WD>(p.weight, 0, c, p.dim, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) b[i] = 0.f;
            if (p.bias != nullptr) load8<WD>(p.bias, 0, c, p.dim, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = fmaf((h[i] - off) * r, w[i], b[i]);
            store8<XD>(p.y, row * p.y_stride + c, p.dim - c, h);
        }
    }
}

// A workgroup takes rows_each rows, its wavefronts every fourth of them where a wavefront takes a row.  NV = 0: a row is read twice and
// dw, db are summed in the plane itself.
template <int XD, int RD, int WD, int T, int NV>
__global__ void __launch_bounds__(threads_of(T))
layer_norm_bwd_kernel(const cc1d_layer_norm_bwd_params p, float *planes, const int64_t rows_each) {
    __shared__ float lds[2][3][16];
    const int lane = T == 64 ? (int)(threadIdx.x & 63) : (int)threadIdx.x, lanes = T == 64 ? 64 : (int)blockDim.x;
    const int wave = threadIdx.x >> 6;
    const int64_t begin = blockIdx.x * rows_each, last = begin + rows_each < p.rows ? begin + rows_each : p.rows;
    const int64_t first = begin + (T == 64 ? wave : 0);
    constexpr int step = T == 64 ? 4 : 1;
    const bool bias = p.dbias != nullptr;
    float *plane = planes + (int64_t)blockIdx.x * (bias ? 2 : 1) * p.dim, *plane_b = plane + p.dim;
    const float over = 1.f / (float)p.dim;
    auto put = [&](int64_t row, int c, const float (&d)[8]) {
        const int n = p.dim - c;
        if (p.dx != nullptr) store8<XD>(p.dx, row * p.dx_stride + c, n, d);
        if (p.dresidual != nullptr) store8<RD>(p.dresidual, row * p.dresidual_stride + c, n, d);
    };
    int turn = 0;                                        // which half of `lds`: a row's sums may still be read when the next one's are written
    // Of a row's differences times r: their own mean `off`, and with n what is left of them the means of w dy and of w dy n.  `sums`: of these differences, of
    // w dy, of the products.
    struct Means { float off, m1, m2; };
    auto means_of = [&](float (&sums)[3]) {
        over_row<T>(sums, lds[turn]);
        turn ^= 1;
        const float off = sums[0] * over;
        return Means{off, sums[1] * over, (sums[2] - off * sums[1]) * over};
    };
    if constexpr (NV > 0) {
        Raw8<WD> wr[NV];
        float w[NV][8], dw[NV][8], db[NV][8];
#pragma unroll
        for (int v = 0; v < NV; ++v) wr[v].load(p.weight, 0, (v * lanes + lane) * 8, p.dim);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            wr[v].to(w[v]);
#pragma unroll
            for (int i = 0; i < 8; ++i) dw[v][i] = db[v][i] = 0.f;
        }
        for (int64_t row = first; row < last; row += step) {
            Raw8<RD, true> hr[NV], dhr[NV];
            Raw8<XD, true> dyr[NV];
            float h[NV][8], dy[NV][8], d[NV][8], sums[3] = {0.f, 0.f, 0.f};
            const float2 st = *reinterpret_cast<const float2 *>(p.stats + 2 * row);
#pragma unroll
            for (int v = 0; v < NV; ++v) hr[v].load(p.h, row * p.h_stride, (v * lanes + lane) * 8, p.dim);
#pragma unroll
            for (int v = 0; v < NV; ++v) dyr[v].load(p.dy, row * p.dy_stride, (v * lanes + lane) * 8, p.dim);
            if (p.dh != nullptr) {
#pragma unroll
                for (int v = 0; v < NV; ++v) dhr[v].load(p.dh, row * p.dh_stride, (v * lanes + lane) * 8, p.dim);
            }
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                hr[v].to(h[v]);
                dyr[v].to(dy[v]);
#pragma unroll
                for (int i = 0; i < 8; ++i) d[v][i] = 0.f;
                if (p.dh != nullptr) dhr[v].to(d[v]);
            }
            // (Behind the row's end dy and w are 0.)
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    h[v][i] = i < p.dim - (v * lanes + lane) * 8 ? (h[v][i] - st.x) * st.y : 0.f;
                    sums[0] += h[v][i];
                    sums[1] += w[v][i] * dy[v][i];
                    sums[2] += (w[v][i] * dy[v][i]) * h[v][i];
                }
            const Means m = means_of(sums);
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int c = (v * lanes + lane) * 8;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float n = h[v][i] - m.off;
                    dw[v][i] += dy[v][i] * n;
                    db[v][i] += dy[v][i];
                    d[v][i] += st.y * ((w[v][i] * dy[v][i] - m.m1) - n * m.m2);
                }
                if (c < p.dim) put(row, c, d[v]);
            }
        }
        if constexpr (T == 64) {                         // the four wavefronts' sums, in their order
            __shared__ float sums[4][NV * 64 * 8];
            auto join = [&](const float (&own)[NV][8], float *to) {
#pragma unroll
                for (int v = 0; v < NV; ++v)
#pragma unroll
                    for (int i = 0; i < 8; ++i) sums[wave][(v * 8 + i) * 64 + lane] = own[v][i];
                lds_barrier();
                for (int k = threadIdx.x; k < NV * 64 * 8; k += 256) {
                    const int c = ((k >> 9) * 64 + (k & 63)) * 8 + ((k >> 6) & 7);
                    if (c < p.dim) to[c] = (sums[0][k] + sums[1][k]) + (sums[2][k] + sums[3][k]);
                }
            };
            join(dw, plane);
            if (bias) {
                lds_barrier();
                join(db, plane_b);
            }
        } else {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int c = (v * lanes + lane) * 8;
                if (c >= p.dim) continue;
                store8<CC1D_F32>(plane, c, p.dim - c, dw[v]);
                if (bias) store8<CC1D_F32>(plane_b, c, p.dim - c, db[v]);
            }
        }
    } else {
        for (int64_t row = first; row < last; row += step) {
            float sums[3] = {0.f, 0.f, 0.f};
            const float2 st = *reinterpret_cast<const float2 *>(p.stats + 2 * row);
            for (int c = lane * 8; c < p.dim; c += lanes * 8) {
                float h[8], dy[8], wv[8];
                load8<RD>(p.h, row * p.h_stride, c, p.dim, h);
                load8<XD>(p.dy, row * p.dy_stride, c, p.dim, dy);
                load8<WD>(p.weight, 0, c, p.dim, wv);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float difference = i < p.dim - c ? (h[i] - st.x) * st.y : 0.f;
                    sums[0] += difference;
                    sums[1] += wv[i] * dy[i];
                    sums[2] += (wv[i] * dy[i]) * difference;
                }
            }
            const Means m = means_of(sums);
            for (int c = lane * 8; c < p.dim; c += lanes * 8) {
                float h[8], dy[8], wv[8], dw[8], db[8], d[8];
                load8<RD>(p.h, row * p.h_stride, c, p.dim, h);
                load8<XD>(p.dy, row * p.dy_stride, c, p.dim, dy);
                load8<WD>(p.weight, 0, c, p.dim, wv);
#pragma unroll
                for (int i = 0; i < 8; ++i) { dw[i] = db[i] = 0.f; d[i] = 0.f; }
                if (row > first) {
                    load8<CC1D_F32>(plane, 0, c, p.dim, dw);
                    if (bias) load8<CC1D_F32>(plane_b, 0, c, p.dim, db);
                }
                if (p.dh != nullptr) load8<RD>(p.dh, row * p.dh_stride, c, p.dim, d);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float n = (h[i] - st.x) * st.y - m.off;
                    dw[i] += dy[i] * n;
                    db[i] += dy[i];
                    d[i] += st.y * ((wv[i] * dy[i] - m.m1) - n * m.m2);
                }
                store8<CC1D_F32>(plane, c, p.dim - c, dw);
                if (bias) store8<CC1D_F32>(plane_b, c, p.dim - c, db);
                put(row, c, d);
            }
        }
    }
}

// Workgroups of the backward on a CU, all of them at once: its registers leave four wavefronts a SIMD, and a workgroup may put its odd one on any
// (16384 rows of 2560: two of five wavefronts 126 us, three 162, the last of them after the others; 8192 of 4096: two of eight 97, one 122).
int bwd_a_cu(int dim) { return 4 / ((bwd_lanes(dim) + 255) / 256); }

}  // namespace
}  // namespace cc1d

using namespace cc1d;

extern "C" {

int cc1d_validate_layer_norm(const cc1d_layer_norm_params *p) {
    if (p == nullptr) return CC1D_ERR_NULL_POINTER;
    if (!dtype_ok(p->x_dtype) || !dtype_ok(p->r_dtype) || !dtype_ok(p->w_dtype)) return CC1D_ERR_DTYPE;
    if ((p->r_dtype != p->x_dtype && p->r_dtype != CC1D_F32) || (p->w_dtype != p->x_dtype && p->w_dtype != CC1D_F32)) return CC1D_ERR_DTYPE;
    if (p->rows < 0 || p->dim < 0) return CC1D_ERR_SHAPE;
    if (p->rows == 0 || p->dim == 0) return CC1D_OK;
    if (p->dim > kLongestRow) return CC1D_ERR_TOO_LARGE;
    if (p->x == nullptr || p->weight == nullptr || p->y == nullptr || (p->residual == nullptr) != (p->h == nullptr)) return CC1D_ERR_NULL_POINTER;
    if (!on_elements(p->x, p->x_dtype) || !on_elements(p->y, p->x_dtype) || !on_elements(p->residual, p->r_dtype) || !on_elements(p->h, p->r_dtype) ||
        !on_elements(p->weight, p->w_dtype) || !on_elements(p->bias, p->w_dtype) || (reinterpret_cast<uintptr_t>(p->stats) & 7u) != 0) return CC1D_ERR_ROW_LAYOUT;
    return CC1D_OK;
}

int cc1d_layer_norm_fwd(const cc1d_layer_norm_params *p, cc1d_stream_t stream) {
    const int st = cc1d_validate_layer_norm(p);
    if (st != CC1D_OK || p->rows == 0 || p->dim == 0) return st;
    return by_types(p->x_dtype, p->r_dtype, p->w_dtype, [&](auto xd, auto rd, auto wd) {
        return by_shape(fwd_shape(p->dim), [&](auto lanes, auto vectors) {
            constexpr int L = decltype(lanes)::value, V = decltype(vectors)::value;
            const int lanes_of_block = L == 64 ? 256 : fwd_shape(p->dim).lanes, rows_of_block = L == 64 ? 4 : 1;
            const int64_t blocks = thread_limit() / lanes_of_block, slice = (blocks > 1 ? blocks : 1) * rows_of_block;
            for (int64_t first = 0; first < p->rows; first += slice) {
                const int64_t last = p->rows - first > slice ? first + slice : p->rows;
                CC1D_LAUNCH((layer_norm_fwd_kernel<decltype(xd)::value, decltype(rd)::value, decltype(wd)::value, L, V>),
                            dim3((uint32_t)((last - first + rows_of_block - 1) / rows_of_block)), dim3(lanes_of_block), 0,
                            static_cast<hipStream_t>(stream), *p, first, last);
                const int st = launch_status();
                if (st != CC1D_OK) return st;
            }
            return (int)CC1D_OK;
        });
    });
}

int cc1d_validate_layer_norm_bwd(const cc1d_layer_norm_bwd_params *p) {
    if (p == nullptr) return CC1D_ERR_NULL_POINTER;
    if (!dtype_ok(p->x_dtype) || !dtype_ok(p->r_dtype) || !dtype_ok(p->w_dtype)) return CC1D_ERR_DTYPE;
    if ((p->r_dtype != p->x_dtype && p->r_dtype != CC1D_F32) || (p->w_dtype != p->x_dtype && p->w_dtype != CC1D_F32)) return CC1D_ERR_DTYPE;
    if (p->rows < 0 || p->dim < 0) return CC1D_ERR_SHAPE;
    if (p->dim == 0) return CC1D_OK;
    if (p->dim > kLongestRowBwd / 2) return CC1D_ERR_TOO_LARGE;           // (both sums lie side by side)
    if (p->dweight == nullptr) return CC1D_ERR_NULL_POINTER;
    if (!on_elements(p->dweight, p->w_dtype) || !on_elements(p->dbias, p->w_dtype)) return CC1D_ERR_ROW_LAYOUT;
    if (p->rows == 0) return CC1D_OK;
    if (p->h == nullptr || p->stats == nullptr || p->weight == nullptr || p->dy == nullptr) return CC1D_ERR_NULL_POINTER;
    if (!on_elements(p->h, p->r_dtype) || !on_elements(p->weight, p->w_dtype) || !on_elements(p->dy, p->x_dtype) || !on_elements(p->dh, p->r_dtype) ||
        !on_elements(p->dx, p->x_dtype) || !on_elements(p->dresidual, p->r_dtype) || (reinterpret_cast<uintptr_t>(p->stats) & 7u) != 0) return CC1D_ERR_ROW_LAYOUT;
    return CC1D_OK;
}

int cc1d_layer_norm_bwd_workspace_bytes(const cc1d_layer_norm_bwd_params *p, size_t *bytes) {
    if (bytes == nullptr) return CC1D_ERR_NULL_POINTER;
    *bytes = 0;
    const int st = cc1d_validate_layer_norm_bwd(p);
    if (st != CC1D_OK || p->dim == 0) return st;
    *bytes = (size_t)bwd_parts(p->rows, bwd_a_cu(p->dim)) * (p->dbias != nullptr ? 2 : 1) * (size_t)p->dim * sizeof(float);
    return CC1D_OK;
}

int cc1d_layer_norm_bwd(const cc1d_layer_norm_bwd_params *p, void *workspace, size_t workspace_bytes, cc1d_stream_t stream) {
    size_t need = 0;
    int st = cc1d_layer_norm_bwd_workspace_bytes(p, &need);
    if (st != CC1D_OK || p->dim == 0) return st;
    if (need > 0 && (workspace == nullptr || !aligned16(workspace) || workspace_bytes < need)) return CC1D_ERR_WORKSPACE;
    const int64_t parts = bwd_parts(p->rows, bwd_a_cu(p->dim));
    const int width = p->dbias != nullptr ? 2 * p->dim : p->dim;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (p->rows > 0) {
        const int64_t each = (p->rows + parts - 1) / parts;
        st = by_types(p->x_dtype, p->r_dtype, p->w_dtype, [&](auto xd, auto rd, auto wd) {
            return by_shape(bwd_shape(p->dim), [&](auto lanes, auto vectors) {
                constexpr int L = decltype(lanes)::value, V = decltype(vectors)::value;
                CC1D_LAUNCH((layer_norm_bwd_kernel<decltype(xd)::value, decltype(rd)::value, decltype(wd)::value, L, V>),
                            dim3((uint32_t)parts), dim3(L == 64 ? 256 : bwd_shape(p->dim).lanes), 0, s, *p, static_cast<float *>(workspace), each);
                return launch_status();
            });
        });
        if (st != CC1D_OK) return st;
    }
    CC1D_LAUNCH(norm_dweight_kernel, dim3((uint32_t)(width + 31) / 32), dim3(1024), 0, s, static_cast<const float *>(workspace), (int)parts, width, (int)p->dim,
                p->dweight, p->dbias, (int)p->w_dtype);
    return launch_status();
}

}  // extern "C"
