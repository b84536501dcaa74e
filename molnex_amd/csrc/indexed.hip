// The indexed linear map: rows multiplied with the weights of their class, ragged groups in one launch.
//
//   y[i] = x[i] W[z[i]]            W (S, K, N): one K x N matrix a class; a row out of range gets zeros
//   gx[i] = g[i] W[z[i]]^T
//   gw[s] = sum over the rows i of class s of x[i]^T g[i]
//
// The rows of a class are found through `order` (row numbers by class, those out of range last) and `class_start`
// (mnx_class_groups): they are read and written in place, with no sorted copy.  The grid is sized for the worst case
// (a partial tile per class) and surplus workgroups leave at once, so nothing synchronises.
//
// Three forms, by type and alignment.
//
// 16-bit rows and columns of whole 16-byte pieces: k_indexed_rows16 and k_indexed_weights16, the loop of tile16.h, whose
// loads go straight to LDS from addresses that the lanes gather.
//
// Others (float32, odd widths): k_indexed_rows and k_indexed_weights.  Both operands pass through registers into LDS, the
// next chunk's loads in flight under this one's products; vectors of 16 bytes at the alignment of one element, so any width
// and row distance will do.  An operand whose sum index is contiguous in memory lies in LDS by rows and is read 16 bytes a
// lane; one whose rows are the sum index (W in the forward, x and g in the weights' gradient) lies as it is in memory too
// and is read with the transposing LDS load.  float32 is split into three bfloat16 parts on the way into LDS, of whose nine
// products the six above 2^-24 are formed, smallest first: a product x w is off by 6 2^-24 |x w| at most, and where a value
// is so small (below 2^-109) that its parts become subnormal, by 2^-133 (|x| + |w|) more.  Infinities and values that
// bfloat16's largest does not reach (within 2^-8 of float32's) make sums of parts NaN; sums that come out infinite or NaN
// are formed again from the values themselves, in the order of the rows, with float32 operations.
//
// Few float32 rows: k_indexed_few, on the vector units.
//
// Sums are float32, results rounded once to their type.  The weights' gradient sums a class's rows in slices of about
// `slice` rows; a class of several leaves partial sums in the workspace, which a second kernel adds in order: the same bits
// every time.
#include "bf16_split.h"
#include "elem.h"
#include "tile16.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace mnx {
namespace {

using namespace tile16;

constexpr int kThreads = 256;
constexpr int kBM = 128;

enum { kForward = 0, kGradX = 1 };

template <int DT>
struct Kind {
    static constexpr int planes = DT == kF32 ? 3 : 1;
    static constexpr int kc = DT == kF32 ? 32 : 64;  // sum indices of a chunk
    static constexpr int vec = DT == kF32 ? 4 : 8;   // elements of 16 bytes
    typedef typename Elem<DT>::T T;
    typedef T Vec __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

// `left` elements of a vector at p; zeros behind them.  (The last vector of a row loaded whole and shifted into place would
// be waited for here: 50k float32 rows of 1024 to 1024 took 1026 us so, 775 as it is.)
template <int DT>
__device__ __forceinline__ f32x4 load_vec(const typename Kind<DT>::T* p, int left) {
    constexpr int V = Kind<DT>::vec;
    typename Kind<DT>::Vec v;
    if (left >= V) {
        v = *reinterpret_cast<const typename Kind<DT>::Vec*>(p);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = e < left ? p[e] : typename Kind<DT>::T(0);
    }
    return __builtin_bit_cast(f32x4, v);
}

// A vector into LDS at element `at` of every plane.
template <int DT>
__device__ __forceinline__ void store_vec(short* lds, int plane, int at, const f32x4& v) {
    if constexpr (DT == kF32) {
        uint32_t p[3][2];
        bf16_split2(v[0], v[1], p[0][0], p[1][0], p[2][0]);
        bf16_split2(v[2], v[3], p[0][1], p[1][1], p[2][1]);
        typedef uint32_t u2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int k = 0; k < 3; ++k) *reinterpret_cast<u2*>(lds + k * plane + at) = u2{p[k][0], p[k][1]};
    } else {
        *reinterpret_cast<f32x4*>(lds + at) = v;
    }
}

// Where element (row, k) of an operand by rows lies in LDS, KC a row: 16-byte pieces permuted so that 16 rows' pieces
// of one k meet every bank once.
template <int KC>
__device__ __forceinline__ int by_rows(int row, int k) {
    const int turn = KC == 64 ? (row >> 1) & 7 : (row >> 2) & 3;
    return row * KC + ((((k >> 3) ^ turn) << 3) | (k & 7));
}
// ... and element (k, col) of one whose rows are the sum index, W columns a row: 4 rows' 64 bytes meet every bank once.
template <int W>
__device__ __forceinline__ int by_sums(int k, int col) {
    const int turn = W == 128 ? (k & 3) << 2 : ((k >> 1) & 1) << 2;
    return k * W + ((((col >> 3) ^ turn) << 3) | (col & 7));
}

// The matrix cores' operand of 32 rows from row0, sum indices k0 to k0 + 15.
template <int KC>
__device__ __forceinline__ short8v read_rows(const short* lds, int row0, int k0) {
    const int lane = threadIdx.x & 63;
    return *reinterpret_cast<const short8v*>(lds + by_rows<KC>(row0 + (lane & 31), k0 + 8 * (lane >> 5)));
}
// ... of 32 columns from col0: the load hands lane l of 16 the four k of column l from four rows of 16 columns.
template <int W>
__device__ __forceinline__ short8v read_sums(const short* lds, int col0, int k0) {
    const int lane = threadIdx.x & 63;
    const int k = k0 + 8 * (lane >> 5) + ((lane & 15) >> 2), col = col0 + (lane & 16) + (lane & 3) * 4;
    const short* q = lds + by_sums<W>(k, col);
    return read_tr(q, q + 4 * W);  // k + 4 turns alike
}

// Which class workgroup `unit` serves, when a class of n rows has units(n) of them: the class, the unit's number in it,
// and the sum of extra(n) over the classes before.  cls = classes if it is surplus.  Every lane of a wavefront takes part.
struct Found {
    int cls, unit, extra;
};
// (Positions and row numbers are kept in [0, rows], whatever the caller's plan holds.)
struct Plan {
    const int32_t* order;
    const int32_t* class_start;
    int32_t rows, classes;
    __device__ __forceinline__ int start(int c) const { return min(max(class_start[c], 0), rows); }
    __device__ __forceinline__ int count(int c) const { return max(start(c + 1) - start(c), 0); }
    __device__ __forceinline__ int row(int at) const { return min(max(order[at], 0), rows - 1); }
};
template <typename U, typename E>
__device__ __forceinline__ Found find_class(const Plan& plan, int classes, int unit, U units, E extra) {
    const int lane = threadIdx.x & 63;
    int before = 0, more = 0;
    for (int base = 0; base < classes; base += 64) {
        const int c = base + lane;
        const int n = c < classes ? plan.count(c) : 0;
        const int mine = c < classes ? units(n) : 0, own = c < classes ? extra(n) : 0;
        int sum = mine, esum = own;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int s = __shfl_up(sum, d), t = __shfl_up(esum, d);
            if (lane >= d) {
                sum += s;
                esum += t;
            }
        }
        const uint64_t past = __ballot(before + sum > unit);
        if (past) {
            const int at = __builtin_ctzll(past);
            return {__builtin_amdgcn_readfirstlane(base + at),
                    __builtin_amdgcn_readfirstlane(unit - before - __shfl(sum - mine, at)),
                    __builtin_amdgcn_readfirstlane(more + __shfl(esum - own, at))};
        }
        before += __shfl(sum, 63);
        more += __shfl(esum, 63);
    }
    return {classes, 0, 0};
}

template <int MT, int NT>
__device__ __forceinline__ void clear_acc(f32x16 (&acc)[MT][NT]) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[m][n][q] = 0.f;
}

// The products of one chunk's 16 sum indices, fragments of every plane read.
template <int DT, int MT, int NT>
__device__ __forceinline__ void multiply(const short8v (&a)[Kind<DT>::planes][MT], const short8v (&b)[Kind<DT>::planes][NT],
                                         f32x16 (&acc)[MT][NT]) {
    constexpr int PA[6] = {2, 1, 0, 1, 0, 0}, PB[6] = {0, 1, 2, 0, 1, 0};
    constexpr int Z = Kind<DT>::planes == 3 ? 6 : 1;
#pragma unroll
    for (int z = 0; z < Z; ++z)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n)
                acc[m][n] = mfma<DT != kF16>(a[Z == 6 ? PA[z] : 0][m], b[Z == 6 ? PB[z] : 0][n], acc[m][n]);
}

struct RowsArgs {
    const void* a;  // x or g: rows of `sums` values, lda apart
    const void* w;
    void* out;      // rows of `cols` values
    int64_t lda;
    Plan plan;
    int32_t sums, cols, col_tiles;
    uint32_t units;
};

// The sum over k < n of float32 values at a(k) and b(k), eight products' loads at a time; NaN as soon as it is.  (50k rows of
// 1024 to 1024 whose every sum overflows take 31 ms forward, 94 with one product at a time.)
template <typename A, typename B>
__device__ __forceinline__ float plain_sum(int n, A a, B b) {
    float sum = 0;
#pragma unroll 1
    for (int k0 = 0; k0 < n && sum == sum; k0 += 8) {
        float x[8], y[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            x[k] = *a(min(k0 + k, n - 1));
            y[k] = *b(min(k0 + k, n - 1));
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k0 + k < n) sum = __builtin_fmaf(x[k], y[k], sum);
    }
    return sum;
}
__device__ __forceinline__ bool finite(float v) { return fabsf(v) < HUGE_VALF; }

// y or gx: BM rows of one class against BN columns.  50k float32 rows of 1024 to 1024 take 772 us forward (136 TFLOP/s of
// float32 products, 815 of the matrix cores') and 656 for gx; 50k of 128 to 128 22 us each way, where the 51 MB of rows
// take 10: splitting into parts and a chunk's wait for the next one bound it.
template <int DT, int DIR, int BM, int BN>
__global__ void __launch_bounds__(kThreads) k_indexed_rows(RowsArgs p) {
    using T = typename Kind<DT>::T;
    constexpr int KC = Kind<DT>::kc, V = Kind<DT>::vec, PL = Kind<DT>::planes;
    constexpr int NA = BM * KC / V / kThreads, NB = BN * KC / V / kThreads;  // vectors a thread
    constexpr int VR = KC / V;       // vectors of a row's chunk
    constexpr int VC = BN / V;       // vectors of a sum index's columns
    constexpr int WM = BM / 2, WN = BN / 2, MT = WM / 32, NT = WN / 32;
    __shared__ short sA[PL * BM * KC], sB[PL * BN * KC];
    __shared__ int32_t rows[BM];
    const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Column tiles of the same rows, and then rows of the same class, side by side on one XCD
    const uint32_t per = (p.units + 7) / 8, u = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (u >= p.units) return;
    const int row_tile = int(u / uint32_t(p.col_tiles)), col0 = int(u % uint32_t(p.col_tiles)) * BN;
    const int classes = p.plan.classes;
    const Found f = find_class(p.plan, classes + 1, row_tile, [](int n) { return (n + BM - 1) / BM; },
                               [](int) { return 0; });
    if (f.cls > classes) return;
    const int first = p.plan.start(f.cls) + f.unit * BM;
    const int count = min(BM, p.plan.start(f.cls + 1) - first);  // at least 1
    for (int i = tid; i < BM; i += kThreads) rows[i] = p.plan.row(first + min(i, count - 1));
    __syncthreads();
    const int K = f.cls == classes ? 0 : p.sums;  // zeros for rows out of range
    const T* W = static_cast<const T*>(p.w) + (f.cls == classes ? 0 : int64_t(f.cls) * p.sums * p.cols);
    const T* A = static_cast<const T*>(p.a);

    const T* arow[NA];
#pragma unroll
    for (int i = 0; i < NA; ++i) arow[i] = A + int64_t(rows[(tid + i * kThreads) / VR]) * p.lda;
    f32x4 va[NA], vb[NB];
    auto load = [&](int k0) {
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int k = k0 + (tid % VR) * V;
            va[i] = load_vec<DT>(arow[i] + k, K - k);
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int it = tid + i * kThreads;
            if constexpr (DIR == kForward) {
                const int k = k0 + it / VC, c = col0 + (it % VC) * V;
                vb[i] = load_vec<DT>(W + int64_t(k) * p.cols + c, k < K ? p.cols - c : 0);
            } else {
                const int c = col0 + it / VR, k = k0 + (it % VR) * V;
                vb[i] = load_vec<DT>(W + int64_t(c) * p.sums + k, c < p.cols ? K - k : 0);
            }
        }
    };
    auto put = [&]() {
#pragma unroll
        for (int i = 0; i < NA; ++i)
            store_vec<DT>(sA, BM * KC, by_rows<KC>((tid + i * kThreads) / VR, (tid % VR) * V), va[i]);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int it = tid + i * kThreads;
            if constexpr (DIR == kForward) store_vec<DT>(sB, BN * KC, by_sums<BN>(it / VC, (it % VC) * V), vb[i]);
            else store_vec<DT>(sB, BN * KC, by_rows<KC>(it / VR, (it % VR) * V), vb[i]);
        }
    };
    f32x16 acc[MT][NT];
    clear_acc(acc);
    const int wm = wave & 1, wn = wave >> 1;
    if (K > 0) load(0);
    for (int k0 = 0; k0 < K; k0 += KC) {
        __syncthreads();
        put();
        __syncthreads();
        if (k0 + KC < K) load(k0 + KC);
#pragma unroll
        for (int ks = 0; ks < KC; ks += 16) {
            short8v a[PL][MT], b[PL][NT];
#pragma unroll
            for (int pl = 0; pl < PL; ++pl) {
#pragma unroll
                for (int m = 0; m < MT; ++m) a[pl][m] = read_rows<KC>(sA + pl * BM * KC, wm * WM + m * 32, ks);
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    b[pl][n] = DIR == kForward ? read_sums<BN>(sB + pl * BN * KC, wn * WN + n * 32, ks)
                                               : read_rows<KC>(sB + pl * BN * KC, wn * WN + n * 32, ks);
            }
            multiply<DT, MT, NT>(a, b, acc);
        }
    }
    // acc[m][n][q]: row 32 m + 8 (q / 4) + 4 half + q % 4, column 32 n + l32 of the wave's tile
    T* out = static_cast<T*>(p.out);
    float sound = 0;  // NaN: some sum is not finite
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            const int r = wm * WM + m * 32 + 8 * (q / 4) + 4 * half + q % 4;
            if (r >= count) continue;
            T* to = out + int64_t(rows[r]) * p.cols;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int c = col0 + wn * WN + n * 32 + l32;
                if (c < p.cols) to[c] = T(acc[m][n][q]);
                if constexpr (DT == kF32) sound = __builtin_fmaf(acc[m][n][q], 0.f, sound);
            }
        }
    if constexpr (DT == kF32) {
        if (sound == 0) return;
#pragma unroll 1
        for (int e = 0; e < MT * NT * 16; ++e) {
            const int q = e / NT % 16, r = wm * WM + e / (NT * 16) * 32 + 8 * (q / 4) + 4 * half + q % 4;
            const int c = col0 + wn * WN + e % NT * 32 + l32;
            if (r >= count || c >= p.cols) continue;
            T* to = out + int64_t(rows[r]) * p.cols + c;
            const T *a = A + int64_t(rows[r]) * p.lda, *w = W + (DIR == kForward ? c : int64_t(c) * p.sums);
            if (!finite(*to))
                *to = plain_sum(K, [=](int k) { return a + k; },
                                [=](int k) { return w + (DIR == kForward ? int64_t(k) * p.cols : k); });
        }
    }
}

constexpr int kFewRows = 16, kFewCols = 32, kFewSums = 512;  // rows and columns of a workgroup, sums of a chunk

// float32 y or gx, up to 16 rows of one class against 32 columns, without the matrix cores: where there are few rows, the
// weights' way from memory is all there is, and a thread has 16 vectors of them on theirs at a time (the tiles above wait
// for each chunk of 32 sums).  Forward: eight threads share a row of W, 128 rows of it at a time; gx: 32 threads share a row
// of W^T.  Sums are float32, 32 shares of each, added in order.  64 rows of 8 classes, 1024 to 1024: 18 us (33.5 MB of
// weights), 43 with tiles; one row 7.1 and 41.
template <int DIR>
__global__ void __launch_bounds__(kThreads) k_indexed_few(RowsArgs p) {
    constexpr int R = kFewRows, KC = kFewSums, LD = KC + 4;
    __shared__ __attribute__((aligned(16))) float sx[R * LD];
    __shared__ int32_t rows[R];
    const int tid = threadIdx.x;
    const uint32_t per = (p.units + 7) / 8, u = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (u >= p.units) return;
    const int row_tile = int(u / uint32_t(p.col_tiles)), col0 = int(u % uint32_t(p.col_tiles)) * kFewCols;
    const int classes = p.plan.classes;
    const Found f = find_class(p.plan, classes + 1, row_tile, [](int n) { return (n + R - 1) / R; }, [](int) { return 0; });
    if (f.cls > classes) return;
    const int first = p.plan.start(f.cls) + f.unit * R;
    const int count = min(R, p.plan.start(f.cls + 1) - first);  // at least 1
    if (tid < R) rows[tid] = p.plan.row(first + min(tid, count - 1));
    const int K = f.cls == classes ? 0 : p.sums;  // zeros for rows out of range
    const float* W = static_cast<const float*>(p.w) + (f.cls == classes ? 0 : int64_t(f.cls) * p.sums * p.cols);
    const float* A = static_cast<const float*>(p.a);
    float* out = static_cast<float*>(p.out);
    typedef float Vec __attribute__((ext_vector_type(4), aligned(4)));
    const bool whole = p.sums % 4 == 0 && (DIR == kGradX || p.cols % 4 == 0);
    // columns 4 * part, sums 4 * turn + 128 i of a chunk
    const int part = DIR == kForward ? tid & 7 : tid >> 5, turn = DIR == kForward ? tid >> 3 : tid & 31;
    auto serve = [&](auto some) {
        constexpr int RR = decltype(some)::value;  // rows, `count` of them in earnest
        f32x4 acc[RR];
#pragma unroll
        for (int r = 0; r < RR; ++r) acc[r] = f32x4{0, 0, 0, 0};
        constexpr int NX = RR * KC / 4 / kThreads;  // vectors of x a thread
        // Every vector is there in full or not at all (`whole`: read without a branch, so that all are on their way at
        // once), or its end is looked at.
        auto load = [&](auto all, int k0, Vec(&w)[KC / 128][4], Vec(&x)[NX]) {
            const auto take = [&](const float* row, int at, int end) {
                if constexpr (decltype(all)::value) {
                    const Vec v = *reinterpret_cast<const Vec*>(row + (at < end ? at : 0));
                    return at < end ? v : Vec{0, 0, 0, 0};
                } else {
                    Vec v = {0, 0, 0, 0};
                    if (at + 4 <= end) {
                        v = *reinterpret_cast<const Vec*>(row + at);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (at + e < end) v[e] = row[at + e];
                    }
                    return v;
                }
            };
#pragma unroll
            for (int i = 0; i < KC / 128; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int k = k0 + 4 * turn + 128 * i + (DIR == kForward ? e : 0);
                    const int c = col0 + 4 * part + (DIR == kForward ? 0 : e);
                    if constexpr (DIR == kForward) w[i][e] = take(W + int64_t(min(k, K - 1)) * p.cols, c, k < K ? p.cols : 0);
                    else w[i][e] = take(W + int64_t(min(c, p.cols - 1)) * p.sums, k, K);
                }
#pragma unroll
            for (int i = 0; i < NX; ++i) {
                const int it = tid + i * kThreads;
                x[i] = take(A + int64_t(rows[it / (KC / 4)]) * p.lda, k0 + it % (KC / 4) * 4, K);
            }
        };
        for (int k0 = 0; k0 < K; k0 += KC) {
            Vec w[KC / 128][4], x[NX];  // forward: of four sums four columns each; gx: of four columns four sums
            if (whole) load(std::true_type(), k0, w, x);
            else load(std::false_type(), k0, w, x);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NX; ++i) {
                const int it = tid + i * kThreads;
                *reinterpret_cast<f32x4*>(sx + it / (KC / 4) * LD + it % (KC / 4) * 4) = f32x4(x[i]);
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < KC / 128; ++i) {
                if (k0 + 128 * i >= K) break;
#pragma unroll
                for (int r = 0; r < RR; ++r) {
                    const f32x4 v = *reinterpret_cast<const f32x4*>(sx + r * LD + 4 * turn + 128 * i);
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[r][c] += v[e] * (DIR == kForward ? w[i][e][c] : w[i][c][e]);
                }
            }
        }
        // 32 shares of every sum: two by two, then by way of LDS
        constexpr int OTHER = DIR == kForward ? 32 : 16;  // the lane whose turn is 4 or 16 on
        const int share = DIR == kForward ? (tid >> 6) * 4 + (turn & 3) : turn & 15;
        float* sums = sx;  // [16][RR][32]
        __syncthreads();
#pragma unroll
        for (int r = 0; r < RR; ++r) {
            f32x4 v;
#pragma unroll
            for (int c = 0; c < 4; ++c) v[c] = acc[r][c] + __shfl_xor(acc[r][c], OTHER);
            if (!(tid & OTHER)) *reinterpret_cast<f32x4*>(sums + (share * RR + r) * kFewCols + 4 * part) = v;
        }
        __syncthreads();
        for (int it = tid; it < RR * kFewCols; it += kThreads) {
            const int r = it / kFewCols, c = it % kFewCols;
            float sum = 0;
#pragma unroll
            for (int s = 0; s < 16; ++s) sum += sums[(s * RR + r) * kFewCols + c];
            if (r < count && col0 + c < p.cols) out[int64_t(rows[r]) * p.cols + col0 + c] = sum;
        }
    };
    __syncthreads();
    if (count <= 4) serve(std::integral_constant<int, 4>());
    else if (count <= 8) serve(std::integral_constant<int, 8>());
    else serve(std::integral_constant<int, 16>());
}

struct WeightArgs {
    const void* x;
    const void* g;
    void* gw;
    float* part;
    int64_t ldx, ldg;
    Plan plan;
    int32_t K, N, kt, nt, slice;
    int32_t places;  // of partial sums
    int32_t joins;   // workgroups' worth of joining them, at most
    uint32_t units;
};

// A class of n rows: its slices, those with partial sums, and the rows of each but the last (about the same in all).
__device__ __forceinline__ int slices(int n, int slice) { return n > slice ? (n + slice - 1) / slice : 1; }
__device__ __forceinline__ int slots(int n, int slice) { return n > slice ? (n + slice - 1) / slice : 0; }
__device__ __forceinline__ int slice_length(int n, int slice) {
    const int count = slices(n, slice);
    return ((n + count - 1) / count + 63) & ~63;
}

// A 128 x BN tile of one class's gradient over one slice of its rows.  50k float32 rows of 1024 to 1024 1330 us (79
// TFLOP/s); 50k of 128 to 128 27 us and 6 for the join: both operands' rows are gathered, split and read transposed.
template <int DT, int BN>
__global__ void __launch_bounds__(kThreads) k_indexed_weights(WeightArgs p) {
    using T = typename Kind<DT>::T;
    constexpr int KC = Kind<DT>::kc, V = Kind<DT>::vec, PL = Kind<DT>::planes;
    constexpr int VA = kBM / V, NA = kBM * KC / V / kThreads, STEP_A = kThreads / VA;
    constexpr int VB = BN / V, NB = BN * KC / V / kThreads, STEP_B = kThreads / VB;
    constexpr int WN = BN / 2, NT = WN / 32;
    __shared__ short sA[PL * kBM * KC], sB[PL * BN * KC];
    const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t per = (p.units + 7) / 8, u = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (u >= p.units) return;
    const uint32_t tiles = uint32_t(p.kt) * uint32_t(p.nt);
    const int slice_at = int(u / tiles), tile = int(u % tiles);
    const int k0 = tile / p.nt * kBM, n0 = tile % p.nt * BN;
    const int slice = p.slice;
    const Found f = find_class(p.plan, p.plan.classes, slice_at, [=](int n) { return slices(n, slice); },
                               [=](int n) { return slots(n, slice); });
    if (f.cls >= p.plan.classes) return;
    const int lo = p.plan.start(f.cls), n_class = p.plan.count(f.cls);
    const bool whole = n_class <= slice;
    if (!whole && f.extra + f.unit >= p.places) return;  // not with a plan of class_groups
    const int length = slice_length(n_class, slice);
    const int begin = lo + f.unit * length, end = lo + min(n_class, (f.unit + 1) * length);
    const T *X = static_cast<const T*>(p.x), *G = static_cast<const T*>(p.g);
    const int acol = (tid % VA) * V, arow = tid / VA, bcol = (tid % VB) * V, brow = tid / VB;

    f32x4 va[NA], vb[NB];
    int ra[NA], rb[NB];
    auto find_rows = [&](int r0) {
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int at = r0 + arow + i * STEP_A;
            ra[i] = at < end ? p.plan.row(at) : -1;
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int at = r0 + brow + i * STEP_B;
            rb[i] = at < end ? p.plan.row(at) : -1;
        }
    };
    auto load = [&]() {
#pragma unroll
        for (int i = 0; i < NA; ++i)
            va[i] = load_vec<DT>(X + int64_t(max(ra[i], 0)) * p.ldx + k0 + acol, ra[i] >= 0 ? p.K - k0 - acol : 0);
#pragma unroll
        for (int i = 0; i < NB; ++i)
            vb[i] = load_vec<DT>(G + int64_t(max(rb[i], 0)) * p.ldg + n0 + bcol, rb[i] >= 0 ? p.N - n0 - bcol : 0);
    };
    f32x16 acc[2][NT];
    clear_acc(acc);
    const int wm = wave & 1, wn = wave >> 1;
    if (begin < end) {
        find_rows(begin);
        load();
        find_rows(begin + KC);
    }
    for (int r0 = begin; r0 < end; r0 += KC) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NA; ++i) store_vec<DT>(sA, kBM * KC, by_sums<kBM>(arow + i * STEP_A, acol), va[i]);
#pragma unroll
        for (int i = 0; i < NB; ++i) store_vec<DT>(sB, BN * KC, by_sums<BN>(brow + i * STEP_B, bcol), vb[i]);
        __syncthreads();
        if (r0 + KC < end) {
            load();
            find_rows(r0 + 2 * KC);
        }
#pragma unroll
        for (int ks = 0; ks < KC; ks += 16) {
            short8v a[PL][2], b[PL][NT];
#pragma unroll
            for (int pl = 0; pl < PL; ++pl) {
#pragma unroll
                for (int m = 0; m < 2; ++m) a[pl][m] = read_sums<kBM>(sA + pl * kBM * KC, wm * 64 + m * 32, ks);
#pragma unroll
                for (int n = 0; n < NT; ++n) b[pl][n] = read_sums<BN>(sB + pl * BN * KC, wn * WN + n * 32, ks);
            }
            multiply<DT, 2, NT>(a, b, acc);
        }
    }
    T* out = static_cast<T*>(p.gw) + int64_t(f.cls) * p.K * p.N;
    float* part = p.part + (whole ? 0 : int64_t(f.extra + f.unit) * p.K * p.N);
    float sound = 0;  // NaN: some sum is not finite
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            const int k = k0 + wm * 64 + m * 32 + 8 * (q / 4) + 4 * half + q % 4;
            if (k >= p.K) continue;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int c = n0 + wn * WN + n * 32 + l32;
                if (c >= p.N) continue;
                if (whole) out[int64_t(k) * p.N + c] = T(acc[m][n][q]);
                else part[int64_t(k) * p.N + c] = acc[m][n][q];
                if constexpr (DT == kF32) sound = __builtin_fmaf(acc[m][n][q], 0.f, sound);
            }
        }
    if constexpr (DT == kF32) {
        if (sound == 0) return;
        float* sums = whole ? out : part;
#pragma unroll 1
        for (int e = 0; e < 2 * NT * 16; ++e) {
            const int q = e / NT % 16, k = k0 + wm * 64 + e / (NT * 16) * 32 + 8 * (q / 4) + 4 * half + q % 4;
            const int c = n0 + wn * WN + e % NT * 32 + l32;
            if (k >= p.K || c >= p.N) continue;
            float* to = sums + int64_t(k) * p.N + c;
            if (!finite(*to))
                *to = plain_sum(end - begin, [=](int i) { return X + int64_t(p.plan.row(begin + i)) * p.ldx + k; },
                                [=](int i) { return G + int64_t(p.plan.row(begin + i)) * p.ldg + c; });
        }
    }
}

// ---------------------------------------------------------------------------
// 16-bit types whose rows and columns come in pieces of 16 bytes
// ---------------------------------------------------------------------------

__device__ const __attribute__((aligned(16))) uint32_t kZeros[4] = {0, 0, 0, 0};

// The tile's values, 32 rows of a wavefront's part at a time by way of LDS: store(row, column, eight values) for all within
// rows x cols, numbered in the tile.
template <int BT, typename Store>
__device__ __forceinline__ void store_tile(short* lds, const Acc<BT>& acc, int rows, int cols, Store store) {
    constexpr int W = BT / 2, MT = W / 32, LD = W + 4, ITEMS = W / 16;
    const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i0 = (wave & 1) * W, j0 = (wave >> 1) * W;
    float* part = reinterpret_cast<float*>(lds) + wave * 32 * LD;
    __syncthreads();  // everyone has read its last operands
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int n = 0; n < MT; ++n)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = acc[m][n][4 * q + e];
                *reinterpret_cast<f32x4*>(part + l32 * LD + 32 * n + 8 * q + 4 * half) = v;
            }
        wave_sync();
#pragma unroll
        for (int it = 0; it < ITEMS; ++it) {
            const int item = it * 64 + lane, r = item / (W / 8), jj = item % (W / 8) * 8;
            const int i = i0 + 32 * m + r, j = j0 + jj;
            if (i >= rows || j >= cols) continue;
            float v[8];
            *reinterpret_cast<f32x4*>(v) = *reinterpret_cast<const f32x4*>(part + r * LD + jj);
            *reinterpret_cast<f32x4*>(v + 4) = *reinterpret_cast<const f32x4*>(part + r * LD + jj + 4);
            store(i, j, v);
        }
        wave_sync();
    }
}

// Eight values at any alignment, of which `count` exist.
template <typename T>
__device__ __forceinline__ void store8(T* to, int count, const float (&v)[8]) {
    typedef T Eight __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    if (count >= 8) {
        Eight o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = T(v[e]);
        *reinterpret_cast<Eight*>(to) = o;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < count) to[e] = T(v[e]);
    }
}

// y or gx, BT rows of one class against BT columns: the loop of tile16.h, rows gathered by the lanes' addresses.  What lies
// past the sum's end is read as zeros from elsewhere; rows and columns past the tile's repeat the last and are not stored.
// 100k bfloat16 rows of 64 classes, 1024 to 2048: 560 us, 750 TFLOP/s, 476 for gx (rows in order are no faster: the
// gather is not what bounds it, the tiles' beginnings and ends are); 20k rows of 512 to 512 22 us, where the 46 MB take 9.
template <int DT, int DIR, int BT>
__global__ void __launch_bounds__(256, BT == 128 ? 2 : 1) k_indexed_rows16(RowsArgs p) {
    using T = typename Elem<DT>::T;
    constexpr int FETCH = BT / 32;
    __shared__ __attribute__((aligned(16))) short lds[lds_numbers(BT)];
    __shared__ int32_t rows[BT];
    const uint32_t u = unit_of_block();
    if (u >= p.units) return;
    const int row_tile = __builtin_amdgcn_readfirstlane(u / uint32_t(p.col_tiles));
    const int col0 = __builtin_amdgcn_readfirstlane(u % uint32_t(p.col_tiles)) * BT;
    const int classes = p.plan.classes;
    const Found f = find_class(p.plan, classes + 1, row_tile, [](int n) { return (n + BT - 1) / BT; }, [](int) { return 0; });
    if (f.cls > classes) return;
    const int first = p.plan.start(f.cls) + f.unit * BT;
    const int count = min(BT, p.plan.start(f.cls + 1) - first);  // at least 1
    for (int i = threadIdx.x; i < BT; i += 256) rows[i] = p.plan.row(first + min(i, count - 1));
    __syncthreads();
    T* out = static_cast<T*>(p.out);
    Acc<BT> acc;
    clear<BT>(acc);
    if (f.cls < classes) {
        const int K = p.sums, cols = p.cols;
        const T* A = static_cast<const T*>(p.a);
        const T* W = static_cast<const T*>(p.w) + int64_t(f.cls) * K * cols;
        const RowPlace in = row_place();
        const T* arow[FETCH];
        uint32_t wrow[FETCH];  // bytes; within a chunk of sums, or from the tile's first column's row
        int wsum[FETCH];
#pragma unroll
        for (int n = 0; n < FETCH; ++n) {
            arow[n] = A + int64_t(rows[in.row + 32 * n]) * p.lda + in.number;
            if constexpr (DIR == kForward) {
                const SumPlace s = sum_place<BT, 1>(n);
                wsum[n] = s.sum;
                wrow[n] = 2 * (uint32_t(s.sum) * uint32_t(cols) + uint32_t(min(col0 + s.number, cols - 8)));
            } else {
                wsum[n] = in.number;
                wrow[n] = 2 * (uint32_t(min(in.row + 32 * n, cols - 1 - col0)) * uint32_t(K) + uint32_t(in.number));
            }
        }
        auto load = [&](int c, int n, short* to) {
            const int k0 = c * kRow;
            const T* w = W + (DIR == kForward ? int64_t(k0) * cols : int64_t(col0) * K + k0);
            if (k0 + kRow <= K) {
                if (n < FETCH) load_lds(arow[n] + k0, to);
                else load_lds(w, wrow[n - FETCH], to);
            } else if (n < FETCH) {
                load_lds(k0 + in.number < K ? static_cast<const void*>(arow[n] + k0) : kZeros, to);
            } else {
                const char* from = reinterpret_cast<const char*>(w) + wrow[n - FETCH];
                load_lds(k0 + wsum[n - FETCH] < K ? static_cast<const void*>(from) : kZeros, to);
            }
        };
        products<BT, 1, false, DIR == kForward, DT == kBF16>(lds, (K + kRow - 1) / kRow, acc, load, [](int) {});
    }
    store_tile<BT>(lds, acc, count, p.cols - col0, [&](int i, int j, const float (&v)[8]) {
        store8(out + int64_t(rows[i]) * p.cols + col0 + j, p.cols - col0 - j, v);
    });
}

constexpr int kJoins = 2048;  // workgroups that join a class's partial sums, at most

constexpr int kIds = 1536;  // rows whose places are in LDS at a time

// A BT x BT tile of one class's gradient over one slice of its rows: both operands by sums, their rows gathered by the
// lanes' addresses; behind the slice's end, zeros from elsewhere.  NEAR: rows lie within 4 GB, and LDS holds how far, so
// that an address is one addition (64-bit products of row numbers take as long as the matrix cores here).  The same 100k
// rows: 483 us, 870 TFLOP/s, the join of partial sums with it.
template <int DT, int BT, bool NEAR>
__global__ void __launch_bounds__(256, BT == 128 ? 2 : 1) k_indexed_weights16(WeightArgs p) {
    using T = typename Elem<DT>::T;
    constexpr int FETCH = BT / 32;
    constexpr uint32_t NONE = ~0u;
    __shared__ __attribute__((aligned(16))) short lds[lds_numbers(BT)];
    __shared__ uint32_t xid[kIds], gid[NEAR ? kIds : 1];  // bytes, or row numbers
    const uint32_t u = unit_of_block();
    if (u >= p.units) return;
    const uint32_t tiles = uint32_t(p.kt) * uint32_t(p.nt);
    const int slice_at = __builtin_amdgcn_readfirstlane(u / tiles);
    const int tile = __builtin_amdgcn_readfirstlane(u % tiles);
    const int tk = tile / p.nt, tn = tile - tk * p.nt;
    const int k0 = __builtin_amdgcn_readfirstlane(tk) * BT, n0 = __builtin_amdgcn_readfirstlane(tn) * BT;
    const int slice = p.slice;
    const Found f = find_class(p.plan, p.plan.classes, slice_at, [=](int n) { return slices(n, slice); },
                               [=](int n) { return slots(n, slice); });
    if (f.cls >= p.plan.classes) return;
    const int lo = p.plan.start(f.cls), n_class = p.plan.count(f.cls);
    const bool whole = n_class <= slice;
    if (!whole && f.extra + f.unit >= p.places) return;  // not with a plan of class_groups
    const int length = slice_length(n_class, slice);
    const int begin = lo + f.unit * length, end = lo + min(n_class, (f.unit + 1) * length);
    const T *X = static_cast<const T*>(p.x), *G = static_cast<const T*>(p.g);
    int sum[FETCH];
    uint32_t xcol[FETCH], gcol[FETCH];  // bytes; the last piece may reach into the rows' padding
#pragma unroll
    for (int n = 0; n < FETCH; ++n) {
        const SumPlace s = sum_place<BT, 1>(n);
        sum[n] = s.sum;
        xcol[n] = 2 * uint32_t(min(k0 + s.number, (p.K - 1) & ~7));
        gcol[n] = 2 * uint32_t(min(n0 + s.number, (p.N - 1) & ~7));
    }
    Acc<BT> acc;
    clear<BT>(acc);
    for (int at = begin; at < end; at += kIds) {
        __syncthreads();
        const int here = min(kIds, end - at);
        for (int i = threadIdx.x; i < kIds; i += 256) {
            const int row = i < here ? p.plan.row(at + i) : 0;
            xid[i] = i < here ? (NEAR ? uint32_t(row) * uint32_t(2 * p.ldx) : uint32_t(row)) : NONE;
            if constexpr (NEAR) gid[i] = uint32_t(row) * uint32_t(2 * p.ldg);
        }
        __syncthreads();
        uint32_t xrow[FETCH], grow[FETCH];
        auto ahead = [&](int c) {
#pragma unroll
            for (int n = 0; n < FETCH; ++n) {
                xrow[n] = xid[c * kRow + sum[n]];
                grow[n] = NEAR ? gid[c * kRow + sum[n]] : xrow[n];
            }
        };
        auto load = [&](int, int n, short* to) {
            const bool of_x = n < FETCH;
            const int m = of_x ? n : n - FETCH;
            const T* base = of_x ? X : G;
            const uint32_t col = of_x ? xcol[m] : gcol[m], row = of_x ? xrow[m] : grow[m];
            const char* from = reinterpret_cast<const char*>(base);
            from += NEAR ? uint64_t(row + col) : uint64_t(row) * uint64_t(2 * (of_x ? p.ldx : p.ldg)) + col;
            load_lds(xrow[m] != NONE ? static_cast<const void*>(from) : kZeros, to);
        };
        products<BT, 1, true, true, DT == kBF16>(lds, (here + kRow - 1) / kRow, acc, load, ahead);
    }
    T* out = static_cast<T*>(p.gw) + int64_t(f.cls) * p.K * p.N;
    float* part = p.part + (whole ? 0 : int64_t(f.extra + f.unit) * p.K * p.N);
    store_tile<BT>(lds, acc, p.K - k0, p.N - n0, [&](int i, int j, const float (&v)[8]) {
        const int64_t at = int64_t(k0 + i) * p.N + n0 + j;
        const int left = p.N - n0 - j;
        if (whole) store8(out + at, left, v);
        else store8(part + at, left, v);
    });
}

// The partial sums of the classes with several slices, added in order: a workgroup takes 128 elements of such a class at a
// time, eight shares of the slices (in order again) of 32 threads each.
template <int DT>
__global__ void __launch_bounds__(kThreads) k_indexed_join(WeightArgs p) {
    using T = typename Elem<DT>::T;
    __shared__ f32x4 share[8][32];
    const int slice = p.slice, classes = p.plan.classes;
    const int64_t size = int64_t(p.K) * p.N;
    const int units = int(min((size + 127) / 128, int64_t(kJoins)));  // of a class
    const int lane = threadIdx.x & 63, col = threadIdx.x & 31, group = threadIdx.x >> 5;
    typedef float Four __attribute__((ext_vector_type(4), aligned(4)));
    for (int u = blockIdx.x; u < p.joins; u += gridDim.x) {
        // the class: of those with several slices, this many come before it
        int ahead = u / units, cls = -1, before = 0;
        for (int base = 0; base < classes && cls < 0; base += 64) {
            const int c = base + lane, n = c < classes ? p.plan.count(c) : 0;
            uint64_t several = __ballot(n > slice);
            const int here = __popcll(several);
            if (ahead < here) {
                for (; ahead > 0; --ahead) several &= several - 1;
                cls = __builtin_ctzll(several);
                before += lane < cls ? slots(n, slice) : 0;
                cls += base;
            } else {
                ahead -= here;
                before += slots(n, slice);
            }
        }
        if (cls < 0) return;
        for (int d = 32; d; d >>= 1) before += __shfl_xor(before, d);
        // (a plan of nonsense may say anything)
        const int count = before >= 0 && before < p.places ? min(slots(p.plan.count(cls), slice), p.places - before) : 0;
        const int each = (count + 7) / 8;
        const float* part = p.part + (count ? before * size : 0);
        T* out = static_cast<T*>(p.gw) + cls * size;
        for (int64_t e0 = int64_t(u % units) * 128; e0 < size; e0 += int64_t(units) * 128) {
            const int64_t e = e0 + col * 4;
            f32x4 sum = {0, 0, 0, 0};
            const int end = min((group + 1) * each, count);
            if (e + 4 <= size) {
#pragma unroll 8
                for (int s = group * each; s < end; ++s) sum += f32x4(*reinterpret_cast<const Four*>(part + s * size + e));
            } else {
                for (int s = group * each; s < end; ++s)
                    for (int k = 0; k < 4; ++k)
                        if (e + k < size) sum[k] += part[s * size + e + k];
            }
            share[group][col] = sum;
            __syncthreads();
            if (group == 0) {
#pragma unroll
                for (int g = 1; g < 8; ++g) sum += share[g][col];
                for (int k = 0; k < 4; ++k)
                    if (e + k < size) out[e + k] = T(sum[k]);
            }
            __syncthreads();
        }
    }
}

int check_shape(const char* what, int64_t rows, int32_t classes, int64_t in, int64_t out, int32_t dtype) {
    MNX_REQUIRE(elem_valid(dtype), "%s: unknown type %d", what, dtype);
    MNX_REQUIRE(rows >= 0 && rows <= (int64_t(1) << 30), "%s: %lld rows", what, (long long)rows);  // slices count in 32 bits
    MNX_REQUIRE(classes >= 1 && classes <= MNX_CLASS_GROUPS_MAX_CLASSES, "%s: 1 to %d classes, got %d", what,
                MNX_CLASS_GROUPS_MAX_CLASSES, classes);
    MNX_REQUIRE(in >= 1 && out >= 1 && in <= MNX_INDEXED_MAX_WIDTH && out <= MNX_INDEXED_MAX_WIDTH,
                "%s: widths of 1 to %d, got %lld and %lld", what, MNX_INDEXED_MAX_WIDTH, (long long)in, (long long)out);
    return MNX_OK;
}

// Whether rows are whole pieces of 16 bytes at multiples of 16 bytes: the loads of tile16.h.  `padded`: the last piece may
// hold what lies between the rows.
inline bool in_pieces(int dtype, const void* p, int64_t ld, int64_t width, bool padded = false) {
    return dtype != kF32 && reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0 &&
           (width % 8 == 0 || (padded && ld == ceil_div(width, 8) * 8));
}

constexpr int64_t kCUs = 256;

template <int DT, int DIR>
int rows_product(RowsArgs p, mnx_stream_t stream) {
    const int64_t rows = p.plan.rows, parts = std::min<int64_t>(rows, p.plan.classes + 1);
    const bool pieces = in_pieces(DT, p.a, p.lda, p.sums) && in_pieces(DT, p.w, p.cols, p.cols) &&
                        in_pieces(DT, p.out, p.cols, p.cols);
    int tile = kBM;
    if (DT != kF32 && pieces) {
        const int64_t wide = ceil_div(rows, 256) * ceil_div(p.cols, 256), few = ceil_div(rows, 128) * ceil_div(p.cols, 128);
        tile = few < kCUs || p.cols <= 64 ? 64 : wide >= 4 * kCUs && p.cols > 128 ? 256 : 128;
    }
    if constexpr (DT == kF32) {
        // 256 rows of 5 classes, 128 to 128, 6.9 us so (104 workgroups), 9.5 with tiles; 2048 rows 12.8 (536) and 9.7; 256
        // rows of 8 classes, 1024 to 1024, 33 (800) and 44; 64 to 64 by tiles always (5.2 us, 6.8 so)
        const int64_t cols = ceil_div(p.cols, kFewCols), units = (rows / kFewRows + parts) * cols;
        if (p.sums > 64 && units <= std::clamp(p.sums, 512, 1024)) {
            p.col_tiles = int32_t(cols);
            p.units = uint32_t(units);
            k_indexed_few<DIR><<<uint32_t(ceil_div(units, 8) * 8), kThreads, 0, stream>>>(p);
            MNX_CHECK_LAUNCH();
            return MNX_OK;
        }
    }
    const int BN = pieces ? tile : p.cols <= 64 ? 64 : 128;
    p.col_tiles = int32_t(ceil_div(p.cols, BN));
    // half the rows each where whole tiles would leave CUs free: 12345 float16 rows of 77 to 333 13.7 us so, 16.7 with 128;
    // 50k float32 rows of 128, which fill them, 25 against 22.5
    if (!pieces && ceil_div(rows, kBM) * p.col_tiles < kCUs) tile = kBM / 2;
    const int64_t units = (rows / tile + parts) * p.col_tiles;
    MNX_REQUIRE(units < (int64_t(1) << 23), "indexed linear: too many rows and columns for one call");
    p.units = uint32_t(units);
    if constexpr (DT != kF32) {
        if (pieces) {
            const auto kernel = tile == 256 ? k_indexed_rows16<DT, DIR, 256>
                                : tile == 128 ? k_indexed_rows16<DT, DIR, 128> : k_indexed_rows16<DT, DIR, 64>;
            kernel<<<uint32_t(ceil_div(units, 128) * 128), kThreads, 0, stream>>>(p);
            MNX_CHECK_LAUNCH();
            return MNX_OK;
        }
    }
    const auto kernel = tile == 64 ? (BN == 64 ? k_indexed_rows<DT, DIR, 64, 64> : k_indexed_rows<DT, DIR, 64, 128>)
                                   : (BN == 64 ? k_indexed_rows<DT, DIR, 128, 64> : k_indexed_rows<DT, DIR, 128, 128>);
    kernel<<<uint32_t(ceil_div(units, 8) * 8), kThreads, 0, stream>>>(p);
    MNX_CHECK_LAUNCH();
    return MNX_OK;
}

// Microseconds, about, of a gradient's tiles where every class has `rows` rows cut into `cuts`.
double weights_time(double rows, double classes, double cuts, double tiles, double slots, double chunk, double ends) {
    return std::max(classes * cuts * tiles / slots, 1.0) * (std::ceil(rows / cuts / 64) * chunk + ends);
}

// Rows of a slice.  More slices than classes reach more of the card where tiles are few, and cost their partial sums
// (8 TB/s, written and read: mostly through the caches).  64 rows take about 8 us by way of registers (float32, odd
// widths), three workgroups a CU, and 1 with tile16.h, two a CU, or 1.6 where one has its CU to itself.  Where classes
// stay whole, those of up to two or four times the average do.
int64_t slice_rows(int64_t rows, int64_t K, int64_t N, int64_t classes, int32_t dtype) {
    const bool registers = dtype == kF32 || ((K % 8 || N % 8) && (K < 384 || N < 384));
    const double tiles = double(ceil_div(K, kBM) * ceil_div(N, kBM)), average = std::max(double(rows) / classes, 1.0);
    double best = 1, least = HUGE_VAL;
    for (double cuts = 1; cuts <= 1024 && (cuts == 1 || average / cuts >= 64); cuts *= 2) {
        const double sums = cuts > 1 ? 2 * classes * cuts * double(K) * double(N) * 4 / 8e6 : 0;
        const double time = registers ? weights_time(average, double(classes), cuts, tiles, 3 * kCUs, 8, 6)
                                      : weights_time(average, double(classes), cuts, tiles, 2 * kCUs,
                                                     classes * cuts * tiles <= kCUs ? 1.6 : 1, 6);
        if (time + sums < least) {
            least = time + sums;
            best = cuts;
        }
    }
    return std::max<int64_t>(ceil_div(int64_t((best > 1 ? 1 : registers ? 2 : 4) * average / best), 64) * 64, 128);
}

// Slices with partial sums, at most: a class of several has at most twice its share of them.
int64_t places(int64_t rows, int64_t classes, int64_t slice) {
    return rows <= slice ? 0 : std::min(2 * (rows / slice), rows / slice + classes);
}

template <int DT>
int weights_product(WeightArgs p, mnx_stream_t stream) {
    const int64_t rows = p.plan.rows;
    const bool pieces = in_pieces(DT, p.x, p.ldx, p.K, true) && in_pieces(DT, p.g, p.ldg, p.N, true);
    int tile = kBM;
    const int64_t parts = rows / p.slice + p.plan.classes;
    if (DT != kF32 && pieces) {
        // tiles of 256 take 1.2 us a chunk and 15 more, one a CU, of 128 0.94 and 6, two a CU
        const double average = double(rows) / p.plan.classes, cuts = std::max(1.0, average / p.slice);
        const auto time = [&](int64_t side, double slots, double chunk, double ends) {
            const double tiles = double(ceil_div(p.K, side) * ceil_div(p.N, side));
            return weights_time(average, p.plan.classes, cuts, tiles, slots, chunk, ends);
        };
        if (time(256, kCUs, 1.2, 15) < time(128, 2 * kCUs, 0.94, 6)) tile = 256;
    }
    const int cols = !pieces && p.N <= 64 ? 64 : tile;
    p.kt = int32_t(ceil_div(p.K, tile));
    p.nt = int32_t(ceil_div(p.N, cols));
    const int64_t units = parts * p.kt * p.nt;
    MNX_REQUIRE(units < (int64_t(1) << 23), "indexed linear: too many classes and columns for one call");
    p.units = uint32_t(units);
    bool done = false;
    if constexpr (DT != kF32) {
        if (pieces) {
            const bool near = std::max(p.ldx, p.ldg) * rows < (int64_t(1) << 31);  // bytes below 2^32
            const auto kernel = near ? (tile == 256 ? k_indexed_weights16<DT, 256, true> : k_indexed_weights16<DT, 128, true>)
                                     : (tile == 256 ? k_indexed_weights16<DT, 256, false> : k_indexed_weights16<DT, 128, false>);
            kernel<<<uint32_t(ceil_div(units, 128) * 128), kThreads, 0, stream>>>(p);
            done = true;
        }
    }
    if (!done) {
        const auto kernel = cols == 64 ? k_indexed_weights<DT, 64> : k_indexed_weights<DT, 128>;
        kernel<<<uint32_t(ceil_div(units, 8) * 8), kThreads, 0, stream>>>(p);
    }
    MNX_CHECK_LAUNCH();
    if (rows > p.slice) {
        // the host does not know how many classes have several slices: workgroups for all that could, 4096 at most (100k rows
        // of 64 classes, 1024 to 2048: 5 us, 32 with a workgroup for each part of every class)
        const int64_t several = std::min<int64_t>(rows / p.slice, p.plan.classes);
        p.joins = int32_t(std::min(ceil_div(int64_t(p.K) * p.N, 128), int64_t(kJoins)) * several);
        k_indexed_join<DT><<<uint32_t(std::min(p.joins, 2 * kJoins)), kThreads, 0, stream>>>(p);
        MNX_CHECK_LAUNCH();
    }
    return MNX_OK;
}

}  // namespace
}  // namespace mnx

using namespace mnx;

extern "C" {

int mnx_indexed_linear(const void* a, int64_t lda, int64_t rows, const int32_t* order, const int32_t* class_start,
                       int32_t classes, const void* weight, int64_t in, int64_t out, int32_t dtype, int32_t transposed,
                       void* result, mnx_stream_t stream) {
    clear_error();
    if (int rc = check_shape("indexed linear", rows, classes, in, out, dtype)) return rc;
    MNX_REQUIRE(lda >= (transposed ? out : in), "indexed linear: rows of %lld values %lld apart",
                (long long)(transposed ? out : in), (long long)lda);
    if (rows == 0) return MNX_OK;
    MNX_REQUIRE(a && order && class_start && weight && result, "indexed linear: null pointer");
    RowsArgs p{a, weight, result, lda, Plan{order, class_start, int32_t(rows), classes},
               int32_t(transposed ? out : in), int32_t(transposed ? in : out), 0, 0};
    const auto go = [&](auto type) {
        constexpr int DT = decltype(type)::value;
        return transposed ? rows_product<DT, kGradX>(p, stream) : rows_product<DT, kForward>(p, stream);
    };
    if (dtype == kF32) return go(std::integral_constant<int, kF32>());
    if (dtype == kBF16) return go(std::integral_constant<int, kBF16>());
    return go(std::integral_constant<int, kF16>());
}

size_t mnx_indexed_linear_wgrad_workspace_bytes(int64_t rows, int32_t classes, int64_t in, int64_t out, int32_t dtype) {
    if (check_shape("indexed linear", rows, classes, in, out, dtype)) return 0;
    return size_t(places(rows, classes, slice_rows(rows, in, out, classes, dtype))) * size_t(in) * size_t(out) *
           sizeof(float);
}

int mnx_indexed_linear_wgrad(const void* x, int64_t ldx, const void* grad, int64_t ldg, int64_t rows,
                             const int32_t* order, const int32_t* class_start, int32_t classes, int64_t in, int64_t out,
                             int32_t dtype, void* grad_weight, void* workspace, size_t workspace_bytes,
                             mnx_stream_t stream) {
    clear_error();
    if (int rc = check_shape("indexed linear", rows, classes, in, out, dtype)) return rc;
    MNX_REQUIRE(ldx >= in && ldg >= out, "indexed linear: rows of %lld and %lld values %lld and %lld apart",
                (long long)in, (long long)out, (long long)ldx, (long long)ldg);
    MNX_REQUIRE(class_start && grad_weight && (rows == 0 || (x && grad && order)), "indexed linear: null pointer");
    const size_t need = mnx_indexed_linear_wgrad_workspace_bytes(rows, classes, in, out, dtype);
    if (need && (!workspace || workspace_bytes < need))
        return set_error(MNX_ERR_WORKSPACE, "indexed linear: workspace too small");
    WeightArgs p{x, grad, grad_weight, static_cast<float*>(workspace), ldx, ldg,
                 Plan{order, class_start, int32_t(rows), classes}, int32_t(in), int32_t(out), 0, 0,
                 int32_t(std::min<int64_t>(slice_rows(rows, in, out, classes, dtype), INT32_MAX / 2)), 0, 0, 0};
    p.places = int32_t(places(rows, classes, p.slice));
    if (dtype == kF32) return weights_product<kF32>(p, stream);
    if (dtype == kBF16) return weights_product<kBF16>(p, stream);
    return weights_product<kF16>(p, stream);
}

}  // extern "C"
