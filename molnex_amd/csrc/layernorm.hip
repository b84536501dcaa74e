// Layer norm over the last axis: forward, backward with the weights' gradients, second order.
//
// Row: mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) r, y = h w + b.  The row's
// derivative is the symmetric matrix J a = r (a - mean(a) - h mean(a h)).
//   backward: gx = J(g w), gw = sum over rows of g h, gb = sum over rows of g
//   second order, seeds u (of gx), p (of gw), q (of gb), with a = g w, alpha = mean(a h), ups = mean(u h):
//     dg = w J u + p h + q,   dw = sum over rows of g J u,
//     dx = J(p g) - r (alpha J u + ups J a) - r h mean(u J a)
// Every sum is in float32; the variance is the mean square about the mean, not a difference of moments.
#include "elem.h"

namespace mnx {

__device__ __forceinline__ float wave_sum(float v) {
    for (int off = 32; off; off >>= 1) v += __shfl_xor(v, off);
    return v;
}

// One wavefront per row, the row read again for each sum.
template <int DT>
__global__ __launch_bounds__(256) void k_ln_fwd(const typename Elem<DT>::T* x, int64_t rows, int width, int64_t ldx,
                                                const void* w, const void* b, int wdt, float eps,
                                                typename Elem<DT>::T* y, float* stats) {
    using T = typename Elem<DT>::T;
    const int lane = threadIdx.x & 63;
    const int64_t row = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    const T* xr = x + row * ldx;
    const float inv = 1.0f / width;
    float s = 0;
    for (int c = lane; c < width; c += 64) s += float(xr[c]);
    const float mu = wave_sum(s) * inv;
    s = 0;
    for (int c = lane; c < width; c += 64) {
        const float d = float(xr[c]) - mu;
        s += d * d;
    }
    const float r = 1.0f / sqrtf(wave_sum(s) * inv + eps);
    for (int c = lane; c < width; c += 64) {
        const float h = (float(xr[c]) - mu) * r;
        y[row * width + c] = T(h * (w ? load_elem(w, c, wdt) : 1.0f) + (b ? load_elem(b, c, wdt) : 0.0f));
    }
    if (lane == 0) {
        stats[row] = mu;
        stats[rows + row] = r;
    }
}

template <int DT>
__global__ __launch_bounds__(256) void k_ln_bwd(const typename Elem<DT>::T* g, int64_t ldg,
                                                const typename Elem<DT>::T* x, int64_t ldx, int64_t rows, int width,
                                                const void* w, int wdt, const float* stats,
                                                typename Elem<DT>::T* gx) {
    using T = typename Elem<DT>::T;
    const int lane = threadIdx.x & 63;
    const int64_t row = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    const T *xr = x + row * ldx, *gr = g + row * ldg;
    const float mu = stats[row], r = stats[rows + row], inv = 1.0f / width;
    float sa = 0, sah = 0;
    for (int c = lane; c < width; c += 64) {
        const float a = float(gr[c]) * (w ? load_elem(w, c, wdt) : 1.0f);
        sa += a;
        sah += a * ((float(xr[c]) - mu) * r);
    }
    sa = wave_sum(sa) * inv;
    sah = wave_sum(sah) * inv;
    for (int c = lane; c < width; c += 64) {
        const float a = float(gr[c]) * (w ? load_elem(w, c, wdt) : 1.0f), h = (float(xr[c]) - mu) * r;
        gx[row * width + c] = T(r * (a - sa - h * sah));
    }
}

// Second order, row part; mean(u) and mean(u h) are left for the column sums.
template <int DT>
__global__ __launch_bounds__(256) void k_ln_bwd2(const typename Elem<DT>::T* g, int64_t ldg,
                                                 const typename Elem<DT>::T* x, int64_t ldx,
                                                 const typename Elem<DT>::T* u, int64_t ldu, int64_t rows, int width,
                                                 const void* w, const void* p, const void* q, int wdt,
                                                 const float* stats, typename Elem<DT>::T* dg,
                                                 typename Elem<DT>::T* dx, float* usums) {
    using T = typename Elem<DT>::T;
    const int lane = threadIdx.x & 63;
    const int64_t row = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    const T *xr = x + row * ldx, *gr = g + row * ldg, *ur = u + row * ldu;
    const float mu = stats[row], r = stats[rows + row], inv = 1.0f / width;
    float sa = 0, sah = 0, su = 0, suh = 0, sua = 0, sb = 0, sbh = 0;
    for (int c = lane; c < width; c += 64) {
        const float gv = gr[c], h = (float(xr[c]) - mu) * r, uv = ur[c];
        const float a = gv * (w ? load_elem(w, c, wdt) : 1.0f), b = p ? gv * load_elem(p, c, wdt) : 0.0f;
        sa += a;
        sah += a * h;
        su += uv;
        suh += uv * h;
        sua += uv * a;
        sb += b;
        sbh += b * h;
    }
    sa = wave_sum(sa) * inv, sah = wave_sum(sah) * inv, su = wave_sum(su) * inv, suh = wave_sum(suh) * inv;
    sua = wave_sum(sua) * inv, sb = wave_sum(sb) * inv, sbh = wave_sum(sbh) * inv;
    const float phi = r * (sua - su * sa - suh * sah);  // mean(u J a)
    for (int c = lane; c < width; c += 64) {
        const float gv = gr[c], h = (float(xr[c]) - mu) * r, uv = ur[c], wv = w ? load_elem(w, c, wdt) : 1.0f;
        const float pv = p ? load_elem(p, c, wdt) : 0.0f, a = gv * wv;
        const float ju = r * (uv - su - h * suh), ja = r * (a - sa - h * sah), jb = r * (gv * pv - sb - h * sbh);
        dg[row * width + c] = T(wv * ju + pv * h + (q ? load_elem(q, c, wdt) : 0.0f));
        dx[row * width + c] = T(jb - r * (sah * ju + suh * ja) - r * h * phi);
    }
    if (lane == 0) {
        usums[row] = su;
        usums[rows + row] = suh;
    }
}

// Column sums over a strip of rows: sum g h and sum g, or (usums given) sum g J u.  partial: (strips, 2, width).
template <int DT>
__global__ __launch_bounds__(256) void k_ln_cols(const typename Elem<DT>::T* g, int64_t ldg,
                                                 const typename Elem<DT>::T* x, int64_t ldx,
                                                 const typename Elem<DT>::T* u, int64_t ldu, int64_t rows, int width,
                                                 const float* stats, const float* usums, float* partial) {
    __shared__ float sums[2][4][64];
    const int lane = threadIdx.x & 63, part = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
    const int64_t strip = (rows + gridDim.y - 1) / gridDim.y, end = min(rows, (blockIdx.y + 1) * strip);
    float s0 = 0, s1 = 0;
    if (c < width)
        for (int64_t row = blockIdx.y * strip + part; row < end; row += 4) {
            const float gv = g[row * ldg + c], r = stats[rows + row], h = (float(x[row * ldx + c]) - stats[row]) * r;
            if (usums) s0 += gv * (r * (float(u[row * ldu + c]) - usums[row] - h * usums[rows + row]));
            else s0 += gv * h, s1 += gv;
        }
    sums[0][part][lane] = s0;
    sums[1][part][lane] = s1;
    __syncthreads();
    if (part < 2 && c < width) {
        const float(&v)[4][64] = sums[part];
        partial[(int64_t(blockIdx.y) * 2 + part) * width + c] = (v[0][lane] + v[1][lane]) + (v[2][lane] + v[3][lane]);
    }
}

__global__ __launch_bounds__(256) void k_ln_cols_join(const float* partial, int strips, int width, int wdt, void* gw,
                                                      void* gb) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= width) return;
    float s0 = 0, s1 = 0;
    for (int s = 0; s < strips; ++s) {
        s0 += partial[int64_t(2 * s) * width + c];
        s1 += partial[int64_t(2 * s + 1) * width + c];
    }
    if (gw) store_elem(gw, c, wdt, s0);
    if (gb) store_elem(gb, c, wdt, s1);
}

static int ln_strips(int64_t rows) { return int(std::max<int64_t>(1, std::min<int64_t>(256, rows / 64))); }

static int ln_check(const char* what, int64_t rows, int64_t width, int dtype, int wdtype) {
    MNX_REQUIRE(elem_valid(dtype) && elem_valid(wdtype), "%s: unknown element type", what);
    MNX_REQUIRE(rows >= 0 && width >= 1 && width <= MNX_LAYER_NORM_MAX_WIDTH, "%s: rows >= 0, 1 <= width <= %d", what,
                MNX_LAYER_NORM_MAX_WIDTH);
    MNX_REQUIRE(rows <= (int64_t(1) << 32), "%s: too many rows", what);
    return MNX_OK;
}

}  // namespace mnx

using namespace mnx;

#define LN_DISPATCH(dtype, CALL)          \
    do {                                  \
        if ((dtype) == kF32) {            \
            constexpr int DT = kF32;      \
            CALL;                         \
        } else if ((dtype) == kBF16) {    \
            constexpr int DT = kBF16;     \
            CALL;                         \
        } else {                          \
            constexpr int DT = kF16;      \
            CALL;                         \
        }                                 \
    } while (0)

extern "C" {

int mnx_layer_norm_fwd(const void* x, int64_t ldx, int64_t rows, int64_t width, const void* weight, const void* bias,
                       double eps, int32_t dtype, int32_t wdtype, void* y, float* stats, mnx_stream_t stream) {
    clear_error();
    if (int rc = ln_check("layer norm", rows, width, dtype, wdtype)) return rc;
    if (rows == 0) return MNX_OK;
    MNX_REQUIRE(x && y && stats && ldx >= width, "layer norm: null pointer or ldx < width");
    LN_DISPATCH(dtype, (k_ln_fwd<DT><<<ceil_div(rows, 4), 256, 0, stream>>>(
                           static_cast<const Elem<DT>::T*>(x), rows, int(width), ldx, weight, bias, wdtype, float(eps),
                           static_cast<Elem<DT>::T*>(y), stats)));
    MNX_CHECK_LAUNCH();
    return MNX_OK;
}

size_t mnx_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t width) {
    Workspace ws{nullptr, 0};
    ws.take<float>(size_t(ln_strips(rows)) * 2 * size_t(std::max<int64_t>(width, 1)));
    ws.take<float>(size_t(std::max<int64_t>(rows, 0)) * 2);
    return ws.used;
}

static int ln_cols(const void* g, int64_t ldg, const void* x, int64_t ldx, const void* u, int64_t ldu, int64_t rows,
                   int64_t width, int dtype, int wdtype, const float* stats, const float* usums, float* partial,
                   void* gw, void* gb, mnx_stream_t stream) {
    const int strips = ln_strips(rows);
    LN_DISPATCH(dtype, (k_ln_cols<DT><<<dim3(ceil_div(width, 64), strips), 256, 0, stream>>>(
                           static_cast<const Elem<DT>::T*>(g), ldg, static_cast<const Elem<DT>::T*>(x), ldx,
                           static_cast<const Elem<DT>::T*>(u), ldu, rows, int(width), stats, usums, partial)));
    MNX_CHECK_LAUNCH();
    k_ln_cols_join<<<ceil_div(width, 256), 256, 0, stream>>>(partial, strips, int(width), wdtype, gw, gb);
    MNX_CHECK_LAUNCH();
    return MNX_OK;
}

int mnx_layer_norm_bwd(const void* grad, int64_t ldg, const void* x, int64_t ldx, int64_t rows, int64_t width,
                       const void* weight, int32_t dtype, int32_t wdtype, const float* stats, void* grad_x,
                       void* grad_weight, void* grad_bias, void* workspace, size_t workspace_bytes,
                       mnx_stream_t stream) {
    clear_error();
    if (int rc = ln_check("layer norm backward", rows, width, dtype, wdtype)) return rc;
    MNX_REQUIRE(rows == 0 || (grad && x && stats && ldg >= width && ldx >= width),
                "layer norm backward: null pointer or a row stride below the width");
    if (rows && grad_x) {
        LN_DISPATCH(dtype, (k_ln_bwd<DT><<<ceil_div(rows, 4), 256, 0, stream>>>(
                               static_cast<const Elem<DT>::T*>(grad), ldg, static_cast<const Elem<DT>::T*>(x), ldx,
                               rows, int(width), weight, wdtype, stats, static_cast<Elem<DT>::T*>(grad_x))));
        MNX_CHECK_LAUNCH();
    }
    if (!grad_weight && !grad_bias) return MNX_OK;
    Workspace ws{static_cast<char*>(workspace), workspace_bytes};
    float* partial = ws.take<float>(size_t(ln_strips(rows)) * 2 * width);
    if (!workspace || !ws.fits()) return set_error(MNX_ERR_WORKSPACE, "layer norm backward: workspace too small");
    return ln_cols(grad, ldg, x, ldx, nullptr, 0, rows, width, dtype, wdtype, stats, nullptr, partial, grad_weight,
                   grad_bias, stream);
}

int mnx_layer_norm_bwd2(const void* grad, int64_t ldg, const void* x, int64_t ldx, const void* seed_x, int64_t ldu,
                        const void* seed_w, const void* seed_b, int64_t rows, int64_t width, const void* weight,
                        int32_t dtype, int32_t wdtype, const float* stats, void* dgrad, void* dx, void* dweight,
                        void* workspace, size_t workspace_bytes, mnx_stream_t stream) {
    clear_error();
    if (int rc = ln_check("layer norm second order", rows, width, dtype, wdtype)) return rc;
    MNX_REQUIRE(rows == 0 || (grad && x && seed_x && stats && dgrad && dx && ldg >= width && ldx >= width &&
                              ldu >= width),
                "layer norm second order: null pointer or a row stride below the width");
    Workspace ws{static_cast<char*>(workspace), workspace_bytes};
    float* partial = ws.take<float>(size_t(ln_strips(rows)) * 2 * width);
    float* usums = ws.take<float>(size_t(rows) * 2);
    if (!workspace || !ws.fits()) return set_error(MNX_ERR_WORKSPACE, "layer norm second order: workspace too small");
    if (rows) {
        LN_DISPATCH(dtype, (k_ln_bwd2<DT><<<ceil_div(rows, 4), 256, 0, stream>>>(
                               static_cast<const Elem<DT>::T*>(grad), ldg, static_cast<const Elem<DT>::T*>(x), ldx,
                               static_cast<const Elem<DT>::T*>(seed_x), ldu, rows, int(width), weight, seed_w, seed_b,
                               wdtype, stats, static_cast<Elem<DT>::T*>(dgrad), static_cast<Elem<DT>::T*>(dx),
                               usums)));
        MNX_CHECK_LAUNCH();
    }
    if (!dweight) return MNX_OK;
    return ln_cols(grad, ldg, x, ldx, seed_x, ldu, rows, width, dtype, wdtype, stats, usums, partial, dweight, nullptr,
                   stream);
}

}  // extern "C"
