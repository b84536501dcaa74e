// Layer norm over the last axis: forward, backward with the weights' gradients, second order.
//
// Row: mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) r, y = h w + b.  The row's
// derivative is the symmetric matrix J a = r (a - mean(a) - h mean(a h)).
//   backward: gx = J(g w), gw = sum over rows of g h, gb = sum over rows of g
//   second order, seeds u (of gx), p (of gw), q (of gb), with a = g w, alpha = mean(a h), ups = mean(u h):
//     dg = w J u + p h + q,   dw = sum over rows of g J u,
//     dx = J(p g) - r (alpha J u + ups J a) - r h mean(u J a)
// Every sum is in float32; the variance is the mean square about the mean, not a difference of moments.
//
// Each array is read or written once, and the bytes bound every kernel here (8 to 40 operations a value): 50,000 x
// 2048 fp32 forward 138 us (6.0 TB/s), backward 208 us (5.9), second order 375 us (5.5); a copy reaches 4.8 TB/s.  A
// row is held in the registers of TPR threads, VPL vectors of four values each: its sums, and then its results, come
// from there.  A workgroup has several such groups of threads, takes rows in turn, and keeps the weights in registers.  The
// backward kernels sum over the rows they take in registers too and leave one partial row of sums a workgroup, which a
// second launch joins, so nothing is read again and the order of the sums is fixed.
#include "elem.h"
#include "wave.h"

namespace mnx {

constexpr int kVec = 4;  // values of a vector

// Vectors are read at the alignment of a value (rows of an odd width start anywhere).
template <int DT>
struct Vec {
    typedef typename Elem<DT>::T T;
    typedef T Packed __attribute__((ext_vector_type(kVec), aligned(sizeof(T))));
};

// Columns c .. c + kVec - 1 of a row of `width` values; 0 past its end.  NT: past the caches.
template <int DT, bool NT = false>
__device__ __forceinline__ typename Vec<DT>::Packed load_raw(const typename Elem<DT>::T* p, int c, int width) {
    typename Vec<DT>::Packed t;
    if (c + kVec <= width) {
        const auto* q = reinterpret_cast<const typename Vec<DT>::Packed*>(p + c);
        if constexpr (NT) t = __builtin_nontemporal_load(q);
        else t = *q;
        return t;
    }
#pragma unroll
    for (int e = 0; e < kVec; ++e) t[e] = c + e < width ? p[c + e] : typename Elem<DT>::T(0.0f);
    return t;
}
template <int DT>
__device__ __forceinline__ void unpack(const typename Vec<DT>::Packed& t, float (&v)[kVec]) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) v[e] = float(t[e]);
}
template <int DT, bool NT = false>
__device__ __forceinline__ void load_vec(const typename Elem<DT>::T* p, int c, int width, float (&v)[kVec]) {
    unpack<DT>(load_raw<DT, NT>(p, c, width), v);
}
template <int DT>
__device__ __forceinline__ void store_vec(typename Elem<DT>::T* p, int c, int width, const float (&v)[kVec]) {
    using T = typename Elem<DT>::T;
    if (c + kVec <= width) {
        typename Vec<DT>::Packed t;
#pragma unroll
        for (int e = 0; e < kVec; ++e) t[e] = T(v[e]);
        // past the caches: 50,000 x 1152 fp32 forward 73 against 92 us, 20,001 x 576 bf16 11.4 against 14.9 us
        __builtin_nontemporal_store(t, reinterpret_cast<typename Vec<DT>::Packed*>(p + c));
    } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e)
            if (c + e < width) p[c + e] = T(v[e]);
    }
}
// The backward kernels' h past the row's end has to be 0, not (0 - mu) r, which may overflow and make a NaN of the
// sums' zeros.  The vectors of a thread that need no test for it: in float16 all, since mu r stays finite; in float32
// those inside the row at every width of the variant, all but the last, or the last two of the widest; in bfloat16
// none, which takes fewer registers (6896 x 2900: 36.6 us, 39.7 without any test; elsewhere within 1 % of that).
template <int DT, int TPR, int VPL>
constexpr int inner_vectors() {
    return DT == kF16 ? VPL : DT == kBF16 ? 0 : TPR == 512 ? VPL / 2 : VPL - 1;
}

// Values of a vector of weights, of the rows' type or float32 (ln_reads); `none` where there is no vector, 0 past the
// end.
template <int DT>
__device__ __forceinline__ void load_weights(const void* p, int c, int width, int dtype, float none,
                                             float (&v)[kVec]) {
    constexpr int V = kVec;
    if (!p) {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = c + e < width ? none : 0.0f;
    } else if (DT == kF32 || dtype == DT) {
        load_vec<DT>(static_cast<const typename Elem<DT>::T*>(p), c, width, v);
    } else {
        load_vec<kF32>(static_cast<const float*>(p), c, width, v);
    }
}

// K sums over the TPR threads of a group, on all of them.  More than a wavefront joins through `lds` (K floats a
// wavefront, two sets used in turn so that one barrier a call suffices; every thread of the workgroup calls it).
template <int TPR, int THREADS, int K>
__device__ __forceinline__ void group_sum(float (&s)[K], float* lds, int& turn) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if constexpr (TPR >= 16) s[k] += dpp_partner<8>(s[k]);
        s[k] += dpp_partner<4>(s[k]);
        s[k] += dpp_partner<2>(s[k]);
        s[k] += dpp_partner<1>(s[k]);
        if constexpr (TPR >= 32) {
            float z = s[k];
            pair_sum_swap16(s[k], z);
        }
        if constexpr (TPR >= 64) {
            float z = s[k];
            pair_sum_swap32(s[k], z);
        }
    }
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        float* set = lds + turn * (THREADS / 64) * K;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) set[(threadIdx.x >> 6) * K + k] = s[k];
        __syncthreads();
        set += threadIdx.x / TPR * W * K;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            s[k] = set[k];
#pragma unroll
            for (int i = 1; i < W; ++i) s[k] += set[i * K + k];
        }
    }
}

template <int DT, int TPR, int VPL, int THREADS>
__global__ __launch_bounds__(THREADS) void k_ln_fwd(const typename Elem<DT>::T* x, int64_t rows, int width,
                                                    int64_t ldx, const void* w, const void* b, int wdt, float eps,
                                                    typename Elem<DT>::T* y, float* stats) {
    constexpr int V = kVec, G = THREADS / TPR;
    __shared__ float lds[2 * THREADS / 64];
    int turn = 0;
    const int t = threadIdx.x % TPR;
    float wv[VPL][V], bv[VPL][V];
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        load_weights<DT>(w, (j * TPR + t) * V, width, wdt, 1.0f, wv[j]);
        load_weights<DT>(b, (j * TPR + t) * V, width, wdt, 0.0f, bv[j]);
    }
    const float inv = 1.0f / width;
    for (int64_t first = int64_t(blockIdx.x) * G; first < rows; first += int64_t(gridDim.x) * G) {
        const int64_t row = first + threadIdx.x / TPR;
        const int here = row < rows ? width : 0;  // a group past the last row reads and stores nothing
        float v[VPL][V], s[1] = {0};
#pragma unroll
        for (int j = 0; j < VPL; ++j) load_vec<DT>(x + row * ldx, (j * TPR + t) * V, here, v[j]);
#pragma unroll
        for (int j = 0; j < VPL; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) s[0] += v[j][e];
        group_sum<TPR, THREADS>(s, lds, turn);
        const float mu = s[0] * inv;
        s[0] = 0;
#pragma unroll
        for (int j = 0; j < VPL; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[j][e] = (j * TPR + t) * V + e < width ? v[j][e] - mu : 0.0f;
                s[0] += v[j][e] * v[j][e];
            }
        group_sum<TPR, THREADS>(s, lds, turn);
        const float r = 1.0f / sqrtf(s[0] * inv + eps);
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
#pragma unroll
            for (int e = 0; e < V; ++e) v[j][e] = v[j][e] * r * wv[j][e] + bv[j][e];
            store_vec<DT>(y + row * width, (j * TPR + t) * V, here, v[j]);
        }
        if (t == 0 && here) {
            stats[row] = mu;
            stats[rows + row] = r;
        }
    }
}

// Sums over the rows that the groups of a workgroup took: `acc` of each thread's columns, joined over the groups into
// row blockIdx.x of partial (.., N, width), or as the results where there is one workgroup.
template <int DT, int TPR, int VPL, int N, int THREADS>
__device__ __forceinline__ void join_groups(const float (&acc)[N][VPL][kVec], float* lds, int width,
                                            float* partial, void* const (&result)[N], int wdt) {
    constexpr int V = kVec, G = THREADS / TPR, C = TPR * V;  // columns of a vector index
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < V; ++e) lds[n * THREADS * V + threadIdx.x * V + e] = acc[n][j][e];
        __syncthreads();
        for (int i = threadIdx.x; i < N * C; i += THREADS) {
            const int n = i / C, c = i % C, col = j * C + c;
            if (col >= width) continue;
            float s = lds[n * THREADS * V + c];
            for (int g = 1; g < G; ++g) s += lds[n * THREADS * V + g * C + c];
            if (gridDim.x > 1) partial[(int64_t(blockIdx.x) * N + n) * width + col] = s;
            else if (result[n]) store_elem(result[n], col, wdt, s);
        }
    }
}

// In 16 bits the next row is on its way, as it lies in memory, while one is worked on: such a row is too short for the
// wavefronts of a compute unit to cover the latency by their number (20,001 x 576 bf16: 25.8 against 31.3 us); in 32
// bits the registers cost more wavefronts than that gains (50,000 x 1152: 172 against 129 us).
template <int DT, int TPR, int VPL, bool NT, int THREADS>
__global__ __launch_bounds__(THREADS) void k_ln_bwd(const typename Elem<DT>::T* g, int64_t ldg,
                                                    const typename Elem<DT>::T* x, int64_t ldx, int64_t rows,
                                                    int width, const void* w, int wdt, const float* stats,
                                                    typename Elem<DT>::T* gx, float* partial, void* gw, void* gb,
                                                    int sums) {
    constexpr int V = kVec, G = THREADS / TPR, kInner = inner_vectors<DT, TPR, VPL>();
    constexpr bool kAhead = DT != kF32;
    extern __shared__ float lds[];
    int turn = 0;
    const int t = threadIdx.x % TPR;
    typename Vec<DT>::Packed nx[VPL], ng[VPL];
    float nmu, nr;
    const auto fetch = [&](int64_t row) {
        const int here = row < rows ? width : 0;  // a group past the last row reads and stores nothing
        nmu = here ? stats[row] : 0.0f;
        nr = here ? stats[rows + row] : 0.0f;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            nx[j] = load_raw<DT, NT>(x + row * ldx, (j * TPR + t) * V, here);
            ng[j] = load_raw<DT, NT>(g + row * ldg, (j * TPR + t) * V, here);
        }
    };
    int64_t first = int64_t(blockIdx.x) * G;
    if constexpr (kAhead) fetch(first + threadIdx.x / TPR);
    float wv[VPL][V], acc[2][VPL][V] = {};
#pragma unroll
    for (int j = 0; j < VPL; ++j) load_weights<DT>(w, (j * TPR + t) * V, width, wdt, 1.0f, wv[j]);
    const float inv = 1.0f / width;
    for (; first < rows; first += int64_t(gridDim.x) * G) {
        const int64_t row = first + threadIdx.x / TPR;
        const int here = row < rows ? width : 0;
        float h[VPL][V], a[VPL][V], s[2] = {0, 0};
        if constexpr (!kAhead) fetch(row);
        const float mu = nmu, r = nr;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            unpack<DT>(nx[j], h[j]);
            unpack<DT>(ng[j], a[j]);
        }
        if constexpr (kAhead) fetch(row + int64_t(gridDim.x) * G);
#pragma unroll
        for (int j = 0; j < VPL; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                h[j][e] = j < kInner || (j * TPR + t) * V + e < width ? (h[j][e] - mu) * r : 0.0f;
                acc[0][j][e] += a[j][e] * h[j][e];
                acc[1][j][e] += a[j][e];
                a[j][e] *= wv[j][e];
                s[0] += a[j][e];
                s[1] += a[j][e] * h[j][e];
            }
        if (!gx) continue;
        group_sum<TPR, THREADS>(s, lds, turn);
        const float sa = s[0] * inv, sah = s[1] * inv;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
#pragma unroll
            for (int e = 0; e < V; ++e) a[j][e] = r * (a[j][e] - sa - h[j][e] * sah);
            store_vec<DT>(gx + row * width, (j * TPR + t) * V, here, a[j]);
        }
    }
    if (sums) join_groups<DT, TPR, VPL, 2, THREADS>(acc, lds, width, partial, {gw, gb}, wdt);
}

// SEEDS: whether there are p and q.  Force matching has neither, and their registers would cost it a wavefront in four
// (20,001 x 576 bf16: 71 against 45 us; 50,000 x 1152 fp32: 275 against 214 us).
template <int DT, int TPR, int VPL, bool SEEDS, bool NT, int THREADS>
__global__ __launch_bounds__(THREADS) void k_ln_bwd2(const typename Elem<DT>::T* g, int64_t ldg,
                                                     const typename Elem<DT>::T* x, int64_t ldx,
                                                     const typename Elem<DT>::T* u, int64_t ldu, int64_t rows,
                                                     int width, const void* w, const void* p, const void* q, int wdt,
                                                     const float* stats, typename Elem<DT>::T* dg,
                                                     typename Elem<DT>::T* dx, float* partial, void* dw, int sums) {
    constexpr int V = kVec, G = THREADS / TPR, kInner = inner_vectors<DT, TPR, VPL>();
    extern __shared__ float lds[];
    int turn = 0;
    const int t = threadIdx.x % TPR;
    float wv[VPL][V], pv[VPL][V], qv[VPL][V], acc[1][VPL][V] = {};
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        load_weights<DT>(w, (j * TPR + t) * V, width, wdt, 1.0f, wv[j]);
        if constexpr (SEEDS) {
            load_weights<DT>(p, (j * TPR + t) * V, width, wdt, 0.0f, pv[j]);
            load_weights<DT>(q, (j * TPR + t) * V, width, wdt, 0.0f, qv[j]);
        }
    }
    const float inv = 1.0f / width;
    for (int64_t first = int64_t(blockIdx.x) * G; first < rows; first += int64_t(gridDim.x) * G) {
        const int64_t row = first + threadIdx.x / TPR;
        const int here = row < rows ? width : 0;  // a group past the last row reads and stores nothing
        float h[VPL][V], gv[VPL][V], uv[VPL][V], s[SEEDS ? 7 : 5] = {};
        const float mu = here ? stats[row] : 0.0f, r = here ? stats[rows + row] : 0.0f;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            load_vec<DT, NT>(x + row * ldx, (j * TPR + t) * V, here, h[j]);
            load_vec<DT, NT>(g + row * ldg, (j * TPR + t) * V, here, gv[j]);
            load_vec<DT, NT>(u + row * ldu, (j * TPR + t) * V, here, uv[j]);
        }
#pragma unroll
        for (int j = 0; j < VPL; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                h[j][e] = j < kInner || (j * TPR + t) * V + e < width ? (h[j][e] - mu) * r : 0.0f;
                const float a = gv[j][e] * wv[j][e];
                s[0] += a;
                s[1] += a * h[j][e];
                s[2] += uv[j][e];
                s[3] += uv[j][e] * h[j][e];
                s[4] += uv[j][e] * a;
                if constexpr (SEEDS) {
                    s[5] += gv[j][e] * pv[j][e];
                    s[6] += gv[j][e] * pv[j][e] * h[j][e];
                }
            }
        group_sum<TPR, THREADS>(s, lds, turn);
        const float sa = s[0] * inv, sah = s[1] * inv, su = s[2] * inv, suh = s[3] * inv, sua = s[4] * inv;
        const float phi = r * (sua - su * sa - suh * sah);  // mean(u J a)
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float hv = h[j][e], gg = gv[j][e];
                const float ju = r * (uv[j][e] - su - hv * suh), ja = r * (gg * wv[j][e] - sa - hv * sah);
                acc[0][j][e] += gg * ju;
                gv[j][e] = wv[j][e] * ju;
                uv[j][e] = -r * (sah * ju + suh * ja + hv * phi);
                if constexpr (SEEDS) {
                    gv[j][e] += pv[j][e] * hv + qv[j][e];
                    uv[j][e] += r * (gg * pv[j][e] - s[5] * inv - hv * (s[6] * inv));
                }
            }
            store_vec<DT>(dg + row * width, (j * TPR + t) * V, here, gv[j]);
            store_vec<DT>(dx + row * width, (j * TPR + t) * V, here, uv[j]);
        }
    }
    if (sums) join_groups<DT, TPR, VPL, 1, THREADS>(acc, lds, width, partial, {dw}, wdt);
}

// Joins the workgroups' sums: partial (parts, N, width).  16 columns a workgroup, each thread every 64th part of one:
// the sums of 512 parts are 8 loads deep, and a narrow row still gives many workgroups.
__global__ __launch_bounds__(1024) void k_ln_join(const float* partial, int parts, int N, int width, int wdt, void* r0,
                                                  void* r1) {
    __shared__ float part[64][16];
    const int c = threadIdx.x & 15, group = threadIdx.x >> 4;
    const int64_t all = int64_t(N) * width, col = int64_t(blockIdx.x) * 16 + c;
    float s = 0;
    if (col < all)
#pragma unroll 8
        for (int i = group; i < parts; i += 64) s += partial[i * all + col];
    part[group][c] = s;
    __syncthreads();
    if (group || col >= all) return;
#pragma unroll
    for (int i = 1; i < 64; ++i) s += part[i][c];
    void* r = col < width ? r0 : r1;
    if (r) store_elem(r, col < width ? col : col - width, wdt, s);
}

// Like load_weights, of any type.
__device__ __forceinline__ void load_any(const void* p, int c, int width, int dtype, float none, float (&v)[kVec]) {
    if (!p) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) v[e] = none;
    } else if (dtype == kF32) load_vec<kF32>(static_cast<const float*>(p), c, width, v);
    else if (dtype == kBF16) load_vec<kBF16>(static_cast<const __bf16*>(p), c, width, v);
    else load_vec<kF16>(static_cast<const _Float16*>(p), c, width, v);
}

// Rows too wide for a workgroup's registers, and weights of a type that load_weights does not read (these kernels read
// any): a workgroup takes a row and reads it again for each sum (from L2: a row is at most a few hundred KB where many
// are in flight), and the column sums are a launch of their own.
//
// Threads of a row: many, so that few rows still have many loads on the way, of a vector each.  2000 x 20,000 fp32:
// forward 75 us (4.3 TB/s), forward with all gradients 252; with 256 threads reading value by value 118 and 366.
// 4 x 70,001: forward 18 us, with those 131.
constexpr int kLnWide = 1024;

template <int DT>
__global__ __launch_bounds__(kLnWide) void k_ln_fwd_wide(const typename Elem<DT>::T* x, int64_t rows, int width,
                                                         int64_t ldx, const void* w, const void* b, int wdt, float eps,
                                                         typename Elem<DT>::T* y, float* stats) {
    constexpr int V = kVec, STEP = kLnWide * V;
    __shared__ float lds[2 * kLnWide / 64];
    int turn = 0;
    const float inv = 1.0f / width;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const auto* xr = x + row * ldx;
        float s[1] = {0}, v[V];
        for (int c = threadIdx.x * V; c < width; c += STEP) {
            load_vec<DT>(xr, c, width, v);
            s[0] += (v[0] + v[1]) + (v[2] + v[3]);
        }
        group_sum<kLnWide, kLnWide>(s, lds, turn);
        const float mu = s[0] * inv;
        s[0] = 0;
        for (int c = threadIdx.x * V; c < width; c += STEP) {
            load_vec<DT>(xr, c, width, v);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = c + e < width ? v[e] - mu : 0.0f;
            s[0] += (v[0] * v[0] + v[1] * v[1]) + (v[2] * v[2] + v[3] * v[3]);
        }
        group_sum<kLnWide, kLnWide>(s, lds, turn);
        const float r = 1.0f / sqrtf(s[0] * inv + eps);
        for (int c = threadIdx.x * V; c < width; c += STEP) {
            float wv[V], bv[V];
            load_vec<DT>(xr, c, width, v);
            load_any(w, c, width, wdt, 1.0f, wv);
            load_any(b, c, width, wdt, 0.0f, bv);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = (v[e] - mu) * r * wv[e] + bv[e];
            store_vec<DT>(y + row * width, c, width, v);
        }
        if (threadIdx.x == 0) {
            stats[row] = mu;
            stats[rows + row] = r;
        }
    }
}

template <int DT>
__global__ __launch_bounds__(kLnWide) void k_ln_bwd_wide(const typename Elem<DT>::T* g, int64_t ldg,
                                                         const typename Elem<DT>::T* x, int64_t ldx, int64_t rows,
                                                         int width, const void* w, int wdt, const float* stats,
                                                         typename Elem<DT>::T* gx) {
    constexpr int V = kVec;
    __shared__ float lds[2 * 2 * kLnWide / 64];
    int turn = 0;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const auto *xr = x + row * ldx, *gr = g + row * ldg;
        const float mu = stats[row], r = stats[rows + row], inv = 1.0f / width;
        float s[2] = {0, 0}, h[V], a[V];
        const auto fetch = [&](int c) {  // h and a = g w, 0 past the end
            float wv[V];
            load_vec<DT>(xr, c, width, h);
            load_vec<DT>(gr, c, width, a);
            load_any(w, c, width, wdt, 1.0f, wv);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                h[e] = c + e < width ? (h[e] - mu) * r : 0.0f;
                a[e] *= wv[e];
            }
        };
        for (int c = threadIdx.x * V; c < width; c += kLnWide * V) {
            fetch(c);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                s[0] += a[e];
                s[1] += a[e] * h[e];
            }
        }
        group_sum<kLnWide, kLnWide>(s, lds, turn);
        const float sa = s[0] * inv, sah = s[1] * inv;
        for (int c = threadIdx.x * V; c < width; c += kLnWide * V) {
            fetch(c);
#pragma unroll
            for (int e = 0; e < V; ++e) a[e] = r * (a[e] - sa - h[e] * sah);
            store_vec<DT>(gx + row * width, c, width, a);
        }
    }
}

// Second order, row part; mean(u) and mean(u h) go to the column sums.
template <int DT>
__global__ __launch_bounds__(kLnWide) void k_ln_bwd2_wide(const typename Elem<DT>::T* g, int64_t ldg,
                                                          const typename Elem<DT>::T* x, int64_t ldx,
                                                          const typename Elem<DT>::T* u, int64_t ldu, int64_t rows,
                                                          int width, const void* w, const void* p, const void* q,
                                                          int wdt, const float* stats, typename Elem<DT>::T* dg,
                                                          typename Elem<DT>::T* dx, float* usums) {
    constexpr int V = kVec;
    __shared__ float lds[2 * 7 * kLnWide / 64];
    int turn = 0;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const auto *xr = x + row * ldx, *gr = g + row * ldg, *ur = u + row * ldu;
        const float mu = stats[row], r = stats[rows + row], inv = 1.0f / width;
        float s[7] = {}, h[V], gv[V], uv[V], wv[V], pv[V];
        const auto fetch = [&](int c) {  // h, g and u, 0 past the end
            load_vec<DT>(xr, c, width, h);
            load_vec<DT>(gr, c, width, gv);
            load_vec<DT>(ur, c, width, uv);
            load_any(w, c, width, wdt, 1.0f, wv);
            load_any(p, c, width, wdt, 0.0f, pv);
#pragma unroll
            for (int e = 0; e < V; ++e) h[e] = c + e < width ? (h[e] - mu) * r : 0.0f;
        };
        for (int c = threadIdx.x * V; c < width; c += kLnWide * V) {
            fetch(c);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float a = gv[e] * wv[e], b = gv[e] * pv[e];
                s[0] += a;
                s[1] += a * h[e];
                s[2] += uv[e];
                s[3] += uv[e] * h[e];
                s[4] += uv[e] * a;
                s[5] += b;
                s[6] += b * h[e];
            }
        }
        group_sum<kLnWide, kLnWide>(s, lds, turn);
        const float sa = s[0] * inv, sah = s[1] * inv, su = s[2] * inv, suh = s[3] * inv, sua = s[4] * inv;
        const float sb = s[5] * inv, sbh = s[6] * inv;
        const float phi = r * (sua - su * sa - suh * sah);  // mean(u J a)
        for (int c = threadIdx.x * V; c < width; c += kLnWide * V) {
            float qv[V];
            fetch(c);
            load_any(q, c, width, wdt, 0.0f, qv);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float ju = r * (uv[e] - su - h[e] * suh), ja = r * (gv[e] * wv[e] - sa - h[e] * sah);
                const float jb = r * (gv[e] * pv[e] - sb - h[e] * sbh);
                gv[e] = wv[e] * ju + pv[e] * h[e] + qv[e];
                uv[e] = jb - r * (sah * ju + suh * ja) - r * h[e] * phi;
            }
            store_vec<DT>(dg + row * width, c, width, gv);
            store_vec<DT>(dx + row * width, c, width, uv);
        }
        if (threadIdx.x == 0) {
            usums[row] = su;
            usums[rows + row] = suh;
        }
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

template <int N>
using Int = std::integral_constant<int, N>;

template <typename F>
static void with_type(int dtype, F&& f) {
    if (dtype == kF32) f(Int<kF32>());
    else if (dtype == kBF16) f(Int<kBF16>());
    else f(Int<kF16>());
}

// A variant by the vectors of a row: threads and vectors a thread that leave few lanes without a value.  A wavefront
// or less a row needs no barrier for its sums, but beyond four vectors a thread its registers leave too few rows on the
// way (50,000 x 2048 fp32 backward: eight vectors 251 us, 256 threads of two 228 us).  Vectors of four values in 16
// bits, too (12,345 x 333 f16 forward: 7.6 us, 8.5 with eight).  Calls f(TPR, VPL) with the two as integral constants; false
// where no variant holds the row.
template <typename F>
static bool ln_variant(int64_t width, F&& f) {
    const int64_t nv = ceil_div(width, kVec);
    if (nv <= 8) return f(Int<8>(), Int<1>()), true;
    if (nv <= 16) return f(Int<16>(), Int<1>()), true;
    if (nv <= 32) return f(Int<32>(), Int<1>()), true;
    if (nv <= 48) return f(Int<16>(), Int<3>()), true;
    if (nv <= 64) return f(Int<64>(), Int<1>()), true;
    if (nv <= 96) return f(Int<32>(), Int<3>()), true;
    if (nv <= 128) return f(Int<64>(), Int<2>()), true;
    if (nv <= 192) return f(Int<64>(), Int<3>()), true;
    if (nv <= 256) return f(Int<64>(), Int<4>()), true;
    if (nv <= 384) return f(Int<128>(), Int<3>()), true;
    if (nv <= 512) return f(Int<256>(), Int<2>()), true;
    if (nv <= 768) return f(Int<256>(), Int<3>()), true;
    if (nv <= 1024) return f(Int<256>(), Int<4>()), true;
    if (nv <= 2048) return f(Int<512>(), Int<4>()), true;
    return false;
}

// Whether load_weights reads the weights.  Other types go to the wide form at any width: asking each vector for its
// type cost the calls that have none of them (700 x 128 fp32 forward 2.92 -> 3.17 us; as a rare branch 2.96, but the
// fp16 backward of 166,666 x 120 31.2 -> 33.4).
static bool ln_reads(int dtype, int wdtype) { return wdtype == dtype || wdtype == kF32; }

constexpr int kLnParts = 512;  // workgroups of the backward kernels at most, so rows of partial sums
constexpr int kLnThreads = 512;  // of their workgroups

// Workgroups of the forward kernel for `need` turns of its groups: what the device holds at once, so that the weights
// are read once a group; but where each would take more than four turns, workgroups of two, whose rows come closer to
// the order of memory (50,000 x 2048 fp32: 138 against 154 us; 20,001 x 576 bf16, 2.4 turns: 13.1 against 12.4).
static int64_t ln_forward_grid(const void* kernel, int threads, int64_t need) {
    const int64_t fill = device_fill_grid(kernel, threads, need);
    return fill > 0 && need > 4 * fill && need <= (int64_t(1) << 24) ? ceil_div(need, 2) : fill;
}

// Whether a backward pass over `arrays` arrays reads past the 256 MB cache: 50,000 x 2048 takes 208 against 226 us so,
// its second order 375 against 390; in 16 bits a lane's loads are narrower and lose by it.
template <int DT>
static bool ln_past_cache(int64_t rows, int64_t width, int arrays) {
    return DT == kF32 && rows * width * arrays * 4 > int64_t(256) << 20;
}

// Strips of rows of the wide form's column sums.
static int ln_strips(int64_t rows) { return int(std::max<int64_t>(1, std::min<int64_t>(256, rows / 64))); }

// Workgroups of a backward kernel whose workgroup takes `groups` rows at a time.
static int64_t ln_parts(const void* kernel, int threads, int64_t rows, int groups) {
    const int64_t need = std::min<int64_t>(std::max<int64_t>(ceil_div(rows, groups), 1), kLnParts);
    return device_fill_grid(kernel, threads, need);
}

constexpr int64_t kLnWideGrid = 1 << 16;

// The backward passes' workspace: the rows of partial sums that the form of this width leaves, and for the wide form's
// column sums two numbers a row.  Rows that fit registers may take either (ln_reads); the wide form's strips are fewer.
struct LnWorkspace : Workspace {
    float *partial, *usums;
    LnWorkspace(void* p, size_t bytes, int64_t rows, int64_t width) : Workspace{static_cast<char*>(p), bytes} {
        const bool held = ln_variant(width, [](auto, auto) {});
        const int64_t parts = held ? std::min<int64_t>(std::max<int64_t>(rows, 1), kLnParts) : ln_strips(rows);
        partial = take<float>(size_t(parts) * 2 * size_t(width));
        usums = take<float>(size_t(rows) * 2);
    }
};

static int ln_check(const char* what, int64_t rows, int64_t width, int dtype, int wdtype) {
    MNX_REQUIRE(elem_valid(dtype) && elem_valid(wdtype), "%s: unknown element type", what);
    MNX_REQUIRE(rows >= 0 && width >= 1 && width <= MNX_LAYER_NORM_MAX_WIDTH, "%s: rows >= 0, 1 <= width <= %d", what,
                MNX_LAYER_NORM_MAX_WIDTH);
    MNX_REQUIRE(rows <= (int64_t(1) << 40), "%s: too many rows", what);
    return MNX_OK;
}

}  // namespace mnx

using namespace mnx;

extern "C" {

int mnx_layer_norm_fwd(const void* x, int64_t ldx, int64_t rows, int64_t width, const void* weight, const void* bias,
                       double eps, int32_t dtype, int32_t wdtype, void* y, float* stats, mnx_stream_t stream) {
    clear_error();
    if (int rc = ln_check("layer norm", rows, width, dtype, wdtype)) return rc;
    if (rows == 0) return MNX_OK;
    MNX_REQUIRE(x && y && stats && ldx >= width, "layer norm: null pointer or ldx < width");
    int64_t grid = 0;
    with_type(dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        using T = typename Elem<DT>::T;
        const T* xs = static_cast<const T*>(x);
        T* ys = static_cast<T*>(y);
        const bool held = ln_reads(dtype, wdtype) && ln_variant(width, [&](auto tpr, auto vpl) {
            constexpr int TPR = decltype(tpr)::value, VPL = decltype(vpl)::value, THREADS = TPR > 256 ? TPR : 256;
            const auto kernel = k_ln_fwd<DT, TPR, VPL, THREADS>;
            grid = ln_forward_grid(reinterpret_cast<const void*>(kernel), THREADS, ceil_div(rows, THREADS / TPR));
            if (grid > 0)
                kernel<<<grid, THREADS, 0, stream>>>(xs, rows, int(width), ldx, weight, bias, wdtype, float(eps), ys,
                                                     stats);
        });
        if (!held) {
            grid = std::min<int64_t>(rows, kLnWideGrid);
            k_ln_fwd_wide<DT><<<grid, kLnWide, 0, stream>>>(xs, rows, int(width), ldx, weight, bias, wdtype, float(eps),
                                                            ys, stats);
        }
    });
    MNX_REQUIRE(grid > 0, "layer norm: device query failed");
    MNX_CHECK_LAUNCH();
    return MNX_OK;
}

size_t mnx_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t width) {
    return LnWorkspace(nullptr, 0, std::max<int64_t>(rows, 0), std::max<int64_t>(width, 1)).used;
}

// `parts` rows of sums in `partial`, joined into the results.
static int ln_join(const float* partial, int64_t parts, int N, int64_t width, int wdtype, void* r0, void* r1,
                   mnx_stream_t stream) {
    k_ln_join<<<ceil_div(N * width, 16), 1024, 0, stream>>>(partial, int(parts), N, int(width), wdtype, r0, r1);
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
    const bool sums = grad_weight || grad_bias;
    if (!sums && (!rows || !grad_x)) return MNX_OK;
    const LnWorkspace ws(workspace, workspace_bytes, rows, width);
    float* partial = ws.partial;
    if (sums && (!workspace || !ws.fits()))
        return set_error(MNX_ERR_WORKSPACE, "layer norm backward: workspace too small");
    int64_t parts = 0;
    bool held = true;
    with_type(dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        using T = typename Elem<DT>::T;
        const T *gs = static_cast<const T*>(grad), *xs = static_cast<const T*>(x);
        T* gx = static_cast<T*>(grad_x);
        held = ln_reads(dtype, wdtype) && ln_variant(width, [&](auto tpr, auto vpl) {
            constexpr int TPR = decltype(tpr)::value, VPL = decltype(vpl)::value, THREADS = kLnThreads;
            const auto kernel = ln_past_cache<DT>(rows, width, 3) ? k_ln_bwd<DT, TPR, VPL, DT == kF32, THREADS>
                                                                  : k_ln_bwd<DT, TPR, VPL, false, THREADS>;
            const size_t lds = size_t(2) * THREADS * kVec * sizeof(float);
            parts = ln_parts(reinterpret_cast<const void*>(kernel), THREADS, rows, THREADS / TPR);
            if (parts > 0)
                kernel<<<parts, THREADS, lds, stream>>>(gs, ldg, xs, ldx, rows, int(width), weight, wdtype, stats, gx,
                                                        partial, grad_weight, grad_bias, sums);
        });
        if (!held) {
            if (rows && gx)
                k_ln_bwd_wide<DT><<<std::min<int64_t>(rows, kLnWideGrid), kLnWide, 0, stream>>>(
                    gs, ldg, xs, ldx, rows, int(width), weight, wdtype, stats, gx);
            parts = ln_strips(rows);
            if (sums)
                k_ln_cols<DT><<<dim3(ceil_div(width, 64), parts), 256, 0, stream>>>(
                    gs, ldg, xs, ldx, nullptr, 0, rows, int(width), stats, nullptr, partial);
        }
    });
    MNX_REQUIRE(parts > 0, "layer norm backward: device query failed");
    MNX_CHECK_LAUNCH();
    if (!sums || (held && parts == 1)) return MNX_OK;
    return ln_join(partial, parts, 2, width, wdtype, grad_weight, grad_bias, stream);
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
    if (!rows && !dweight) return MNX_OK;
    const LnWorkspace ws(workspace, workspace_bytes, rows, width);
    float *partial = ws.partial, *usums = ws.usums;
    if (!workspace || !ws.fits()) return set_error(MNX_ERR_WORKSPACE, "layer norm second order: workspace too small");
    int64_t parts = 0;
    bool held = true;
    with_type(dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        using T = typename Elem<DT>::T;
        const T *gs = static_cast<const T*>(grad), *xs = static_cast<const T*>(x), *us = static_cast<const T*>(seed_x);
        T *dg = static_cast<T*>(dgrad), *dxs = static_cast<T*>(dx);
        held = ln_reads(dtype, wdtype) && ln_variant(width, [&](auto tpr, auto vpl) {
            constexpr int TPR = decltype(tpr)::value, VPL = decltype(vpl)::value, THREADS = kLnThreads;
            auto kernel = k_ln_bwd2<DT, TPR, VPL, false, false, THREADS>;
            if (seed_w || seed_b) kernel = k_ln_bwd2<DT, TPR, VPL, true, false, THREADS>;
            else if (ln_past_cache<DT>(rows, width, 5)) kernel = k_ln_bwd2<DT, TPR, VPL, false, DT == kF32, THREADS>;
            const size_t lds = size_t(THREADS) * kVec * sizeof(float);
            parts = ln_parts(reinterpret_cast<const void*>(kernel), THREADS, rows, THREADS / TPR);
            if (parts > 0)
                kernel<<<parts, THREADS, lds, stream>>>(gs, ldg, xs, ldx, us, ldu, rows, int(width), weight, seed_w,
                                                        seed_b, wdtype, stats, dg, dxs, partial, dweight, !!dweight);
        });
        if (!held) {
            if (rows)
                k_ln_bwd2_wide<DT><<<std::min<int64_t>(rows, kLnWideGrid), kLnWide, 0, stream>>>(
                    gs, ldg, xs, ldx, us, ldu, rows, int(width), weight, seed_w, seed_b, wdtype, stats, dg, dxs, usums);
            parts = ln_strips(rows);
            if (dweight)
                k_ln_cols<DT><<<dim3(ceil_div(width, 64), parts), 256, 0, stream>>>(
                    gs, ldg, xs, ldx, us, ldu, rows, int(width), stats, usums, partial);
        }
    });
    MNX_REQUIRE(parts > 0, "layer norm second order: device query failed");
    MNX_CHECK_LAUNCH();
    if (!dweight || (held && parts == 1)) return MNX_OK;
    // the wide form leaves (strips, 2, width) with the sums in the first half
    return ln_join(partial, parts, held ? 1 : 2, width, wdtype, dweight, nullptr, stream);
}

}  // extern "C"
