// Orthogonalised updates: the Newton-Schulz iteration of many matrices at once, and the Muon step around it.
//
//   m = m + (1 - mu) (g - m),  u = g + mu (m - g) with Nesterov's form, m without     (g negated to maximise)
//   X = u / max(|u|, eps), the Frobenius norm; transposed where it has more rows than columns: X is r x c, r <= c
//   steps times:  A = X X^T,  B = b A + c A A,  X = a X + B X
//   p = (1 - lr wd) p - lr s X,  s by the matrix's shape
//
// Numbers: whatever the matrices' type, every number of X, A and B is a pair hi + lo of float16 scaled by powers of two, in
// the workspace or in LDS, multiplied on the matrix cores with float32 sums.  Their entries are bounded by the iteration
// itself (|X|_2 <= max p(s) over the singular values that can occur, about 1.2 with the usual coefficients), so one scale
// a step, chosen on the host from the coefficients, keeps them inside float16's range.  A pair's rounding is half a step of
// lo, 2^-22 at most and 2e-8 in the mean (float32's own: 2^-24 and 2e-8 to 3e-8), and a product is the three sums lo hi +
// hi lo + hi hi, in this order (lo lo is below 2^-22, 2e-8 in the mean): against float64 the results of float32 matrices are
// about as far off as with torch's float32 products (8192 x 4096: 2.3e-6 of the norm, 3.5e-6 there; 64 x 64: 0.6e-6 to
// 2.4e-6, 1.0e-6 there).  The first X is u itself times a power of two; what remains of 1 / |u| (a factor from 1 to 2) goes
// into the first step's sums.  Results in bfloat16 and float16 are the float32 ones rounded.  A single float16 a number (11
// bits, a third of the products) is not enough for them: a float16 result of 333 x 1234 was off by 1.2e-3 so, six times its
// rounding, and a bfloat16 one of 8192 x 4096 by 8.5e-4 beside a rounding of 1.7e-3.
//
// All matrices of a call share each launch; a table in the workspace, written by a first small kernel from its
// arguments, tells a workgroup its matrix and tile.  Matrices with a side of at most 128 whose X and A fit LDS take one
// workgroup each and one launch for the whole step (k_muon_small).  The others go by way of the workspace, three products a
// step (k_muon_product, by the loop of tile16.h), their rows and columns padded with zeros to multiples of 128, so that
// chunks of the sums are whole; a last tile may reach further, and stores nothing there.  A and B are symmetric: only
// tiles on and below the diagonal are formed, each stored twice.  How a matrix is multiplied goes by its own sizes, and
// sums run in the same order in tiles of every size: a list's results are each matrix's own, bit by bit.
#include "elem.h"
#include "tile16.h"

#include <cmath>
#include <numeric>
#include <type_traits>
#include <vector>

namespace mnx {
namespace {

using namespace tile16;

typedef _Float16 half4 __attribute__((ext_vector_type(4)));

constexpr int kPad = 128;  // sides of the padded matrices are multiples of it
constexpr int kChunk = 4096;  // elements of a matrix that a workgroup of the momentum kernel takes
constexpr int kCast = 64;     // side of the cast kernel's tiles
constexpr int kTableArgs = 34;

// One tensor: `batch` matrices of rows x cols.
struct Mat {
    void* p;         // parameters, or where the orthogonalised matrices go
    const void* g;   // gradients, or the matrices to orthogonalise
    float* m;        // momenta, or null
    _Float16* x[2];  // [batch][rp][cp] pairs: 16 hi, then their 16 lo, along a row
    _Float16* a;     // [batch][rp][rp]
    _Float16* b;
    int32_t rows, cols, r, c, rp, cp, batch, dtype;
    float adjust;    // s
    uint32_t stat0;  // the first matrix's place among the norms
    uint32_t chunk0, cast0, sym0, upd0;  // first workgroup of each kind
};
// what follows a tensor's own units: entry `count` of each prefix
struct Prefix {
    uint32_t chunk, cast, sym, upd;
};

struct __attribute__((aligned(16))) TableArgs {
    Mat mat[kTableArgs];
    int count, first;
};
static_assert(sizeof(TableArgs) <= 3840, "4 KB of arguments");
static_assert(sizeof(Mat) % 16 == 0 && kTableArgs * sizeof(Mat) <= 256 * 16, "16 bytes a thread");

__global__ void __launch_bounds__(256) k_muon_table(TableArgs t, Mat* __restrict__ table) {
    typedef uint32_t Piece __attribute__((ext_vector_type(4)));
    if (threadIdx.x < t.count * (sizeof(Mat) / 16))
        reinterpret_cast<Piece*>(table + t.first)[threadIdx.x] = reinterpret_cast<const Piece*>(t.mat)[threadIdx.x];
}

// The last tensor whose first unit is not past `unit`; FIELD is a member of Mat.
__device__ __forceinline__ int find_mat(const Mat* __restrict__ table, int count, uint32_t Mat::*field, uint32_t unit) {
    int at = 0;
    for (int base = 0; base < count; base += 64) {
        const int i = base + int(threadIdx.x & 63);
        at += __popcll(__ballot(i < count && table[i].*field <= unit));
    }
    return __builtin_amdgcn_readfirstlane(at - 1);
}

struct Momentum {
    float mu, w;     // w = 1 - mu
    int nesterov, maximize;
};

struct Stat {
    int exponent;  // X is stored as u 2^exponent
    float rho;     // X = (u 2^exponent) 2^-12 rho; the first step's sums take rho
};

// u, from the gradient and the momentum after this step.
__device__ __forceinline__ float direction(float g, float m, const Momentum& h) {
    return h.nesterov ? __builtin_fmaf(h.mu, m, h.w * g) : m;
}

// Four consecutive elements, at the alignment of one; `left` of them exist, the others are 0 and not stored.
template <typename T>
__device__ __forceinline__ void load4(const T* p, int64_t left, float (&v)[4]) {
    typedef T Four __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    if (left >= 4) {
        const Four t = *reinterpret_cast<const Four*>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = float(t[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = e < left ? float(p[e]) : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, int64_t left, const float (&v)[4]) {
    typedef T Four __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    if (left >= 4) {
        Four t;
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = T(v[e]);
        *reinterpret_cast<Four*>(p) = t;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < left) p[e] = T(v[e]);
    }
}
template <typename F>
__device__ __forceinline__ void by_type(int dtype, F f) {
    if (dtype == kF32) f(float{});
    else if (dtype == kBF16) f(__bf16{});
    else f(_Float16{});
}

// Momenta, and a partial sum of squares for each chunk of a matrix (float64: squares of any float32).  Bound by bytes: a
// stack of 64 bfloat16 matrices of 512 x 1024, 65 us for 336 MB (5.2 TB/s).
__global__ void __launch_bounds__(256) k_muon_momentum(const Mat* __restrict__ table, int count, Momentum h,
                                                       double* __restrict__ partial) {
    const uint32_t unit = blockIdx.x;
    const int at = find_mat(table, count, &Mat::chunk0, unit);
    const Mat& t = table[at];
    const int64_t n = int64_t(t.rows) * t.cols;
    const uint32_t per = uint32_t((n + kChunk - 1) / kChunk), u = unit - t.chunk0;
    const uint32_t which = u / per;
    const int64_t lo = int64_t(u - which * per) * kChunk, off = which * n;
    double sum = 0;
    by_type(t.dtype, [&](auto type) {
        const auto* g = static_cast<const decltype(type)*>(t.g) + off;
        float v[kChunk / 1024][4], m[kChunk / 1024][4];
#pragma unroll
        for (int k = 0; k < kChunk / 1024; ++k) {
            const int64_t i = lo + k * 1024 + threadIdx.x * 4;
            load4(g + i, n - i, v[k]);
            if (t.m) load4(t.m + off + i, n - i, m[k]);
        }
#pragma unroll
        for (int k = 0; k < kChunk / 1024; ++k) {
            const int64_t i = lo + k * 1024 + threadIdx.x * 4;
            if (t.m) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (h.maximize) v[k][e] = -v[k][e];
                    m[k][e] = __builtin_fmaf(h.mu, m[k][e], h.w * v[k][e]);
                    v[k][e] = direction(v[k][e], m[k][e], h);
                }
                store4(t.m + off + i, n - i, m[k]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += double(v[k][e]) * double(v[k][e]);
        }
    });
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    __shared__ double part[4];
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) partial[unit] = (part[0] + part[1]) + (part[2] + part[3]);
}

// X = (u 2^exponent) 2^-12 rho for a matrix of this norm.
__device__ __forceinline__ Stat stat_of(double norm, double eps) {
    Stat s{0, 1.0f};
    if (!(norm < HUGE_VAL)) s.rho = __builtin_nanf("");  // infinite or NaN somewhere: so is every result
    else if (norm > 0) {
        int e;
        frexp(norm, &e);  // norm = f 2^e, 1/2 <= f < 1
        s.exponent = 12 - e;
        s.rho = float(ldexp(1.0, 12 - s.exponent) / fmax(norm, eps));  // 1 to 2 for a norm of eps or more
    }
    return s;
}

// The norm of each matrix: a workgroup a matrix.
__global__ void __launch_bounds__(256) k_muon_norm(const Mat* __restrict__ table, int count,
                                                   const double* __restrict__ partial, double eps,
                                                   Stat* __restrict__ stats) {
    const int at = find_mat(table, count, &Mat::stat0, blockIdx.x);
    const Mat& t = table[at];
    const uint32_t per = uint32_t((int64_t(t.rows) * t.cols + kChunk - 1) / kChunk);
    const double* mine = partial + t.chunk0 + uint64_t(blockIdx.x - t.stat0) * per;
    double sum = 0;
    for (uint32_t i = threadIdx.x; i < per; i += 256) sum += mine[i];
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    __shared__ double part[4];
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) stats[blockIdx.x] = stat_of(sqrt((part[0] + part[1]) + (part[2] + part[3])), eps);
}

constexpr int kPair = 2;  // numbers of a pair

// Where column j's hi of a row lies; its lo is 16 behind.
__device__ __forceinline__ int place(int j) { return ((j & ~15) << 1) | (j & 15); }

__device__ __forceinline__ void put4(_Float16* to, int64_t plane, const float (&v)[4]) {
    half4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        hi[e] = _Float16(v[e]);
        lo[e] = _Float16(v[e] - float(hi[e]));
    }
    *reinterpret_cast<half4*>(to) = hi;
    *reinterpret_cast<half4*>(to + plane) = lo;
}

// u in the products' layout, zeros around it: bytes again, transposed by way of LDS where matrices are tall.
__global__ void __launch_bounds__(256) k_muon_cast(const Mat* __restrict__ table, int count, Momentum h,
                                                   const Stat* __restrict__ stats) {
    __shared__ float tile[kCast][kCast + 1];
    const int at = find_mat(table, count, &Mat::cast0, blockIdx.x);
    const Mat& t = table[at];
    const int nr = t.rp / kCast, nc = t.cp / kCast;
    uint32_t u = blockIdx.x - t.cast0;
    const uint32_t which = u / uint32_t(nr * nc);
    u -= which * uint32_t(nr * nc);
    const int r0 = int(u / nc) * kCast, c0 = int(u % nc) * kCast;
    const int64_t off = int64_t(which) * t.rows * t.cols;
    const Stat s = stats[t.stat0 + which];
    const bool tall = t.rows > t.cols;
    const int i0 = tall ? c0 : r0, j0 = tall ? r0 : c0;  // of the tensor's own rows and columns
    const int row = threadIdx.x / 16, col = threadIdx.x % 16 * 4;
    _Float16* x = t.x[0] + kPair * (int64_t(which) * t.rp * t.cp + int64_t(r0) * t.cp);
    float v[4][4], m[4][4];
    by_type(t.dtype, [&](auto type) {
        const auto* g = static_cast<const decltype(type)*>(t.g) + off;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = i0 + row + 16 * k, left = i < t.rows ? t.cols - j0 - col : 0;
            const int64_t e = int64_t(i) * t.cols + j0 + col;
            load4(g + e, left, v[k]);
            if (t.m) load4(t.m + off + e, left, m[k]);
        }
    });
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (t.m) v[k][e] = direction(h.maximize ? -v[k][e] : v[k][e], m[k][e], h);
            v[k][e] = ldexpf(v[k][e], s.exponent);
            if (tall) tile[row + 16 * k][col + e] = v[k][e];
        }
        if (!tall) put4(x + kPair * int64_t(row + 16 * k) * t.cp + place(c0 + col), 16, v[k]);
    }
    if (!tall) return;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[k][e] = tile[col + e][row + 16 * k];
        put4(x + kPair * int64_t(row + 16 * k) * t.cp + place(c0 + col), 16, v[k]);
    }
}

// ---------------------------------------------------------------------------
// Products
// ---------------------------------------------------------------------------

enum { kGram = 0, kPoly = 1, kUpdate = 2, kFinal = 3 };

struct Step {
    float own, prod;  // result = own E + prod (product), E the element at the result's place
    int from;         // which X is read
    int first;        // the first step: rho counts
};

struct Apply {
    float lr;
    const float* lr_device;
    float wd, inv;  // inv: of X's scale
};

__device__ __forceinline__ f32x16 mfma(const half8& a, const half8& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// A parameter after its step from what decay leaves of it, in the same float32 operations whatever its type: without the
// empty statement a float16 one would be rounded from the unrounded sum.
__device__ __forceinline__ float stepped(float left, float v, float rate) {
    float sum = __builtin_fmaf(-rate, v, left);
    asm("" : "+v"(sum));
    return sum;
}

template <typename T>
struct Eight {
    typedef T V __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};
// Eight consecutive parameters (or results) from p on, of which `count` exist; `old` holds what is there if all do.
template <typename T>
__device__ __forceinline__ void apply(T* p, int count, const typename Eight<T>::V& old, float decay, float rate,
                                      const float (&v)[8]) {
    if (count >= 8) {
        typename Eight<T>::V o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = T(stepped(decay != 0 ? decay * float(old[e]) : 0.f, v[e], rate));
        *reinterpret_cast<typename Eight<T>::V*>(p) = o;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < count) p[e] = T(stepped(decay != 0 ? decay * float(p[e]) : 0.f, v[e], rate));
    }
}

__device__ __forceinline__ void put8(_Float16* to, const float (&v)[8]) {
    half8 hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        hi[e] = _Float16(v[e]);
        lo[e] = _Float16(v[e] - float(hi[e]));
    }
    *reinterpret_cast<half8*>(to) = hi;
    *reinterpret_cast<half8*>(to + 16) = lo;
}

// A BT x BT tile of one product, the sum over k of I[i][k] J[j][k] (rows of both in memory), or with TR of I[i][k] J[k][j].
//
// The last tile of a row or column may reach past the padded matrix: it reads what lies behind it in the workspace (rows
// and columns of the result that are not stored) and stores none of that.
//
// Tiles of 256, one a CU, are bound by the matrix cores (a matrix of 8192 x 4096: 640 us for the three products of B X, 1.29
// PFLOP/s, 5.8 ms in all; a large library product of as many numbers reaches 1.41 here); those of 192 (366 us for A) and
// 128 by their reads of LDS.  Where a call has fewer tiles than CUs, tiles of 64 and the six chunks they have on their way,
// 6 to 12 us a launch, 15 launches one after the other.
template <int MODE, int BT>
__global__ void __launch_bounds__(256, BT == 128 ? 2 : 1) k_muon_product(const Mat* __restrict__ table, int count,
                                                                        uint32_t units, Step s,
                                                                        const Stat* __restrict__ stats, Apply ap) {
    constexpr bool SYM = MODE == kGram || MODE == kPoly, TR = !SYM;
    constexpr int W = BT / 2, MT = W / 32;  // a wavefront's part
    constexpr int FETCH = BT / 32;
    __shared__ __attribute__((aligned(16))) short lds[lds_numbers(BT)];
    const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = wave & 1, wj = wave >> 1;
    uint32_t u = unit_of_block();
    if (u >= units) return;
    const int at = find_mat(table, count, SYM ? &Mat::sym0 : &Mat::upd0, u);
    const Mat& t = table[at];
    u -= SYM ? t.sym0 : t.upd0;
    const int ni = (t.rp + BT - 1) / BT, nj = (t.cp + BT - 1) / BT;
    const uint32_t tiles = SYM ? uint32_t(ni * (ni + 1) / 2) : uint32_t(ni * nj);
    const uint32_t which = __builtin_amdgcn_readfirstlane(u / tiles);
    u -= which * tiles;
    int ti, tj;
    if (SYM) {
        ti = int((sqrtf(8.0f * float(u) + 1.0f) - 1.0f) * 0.5f);
        while (uint32_t(ti * (ti + 1) / 2) > u) --ti;
        while (uint32_t((ti + 1) * (ti + 2) / 2) <= u) ++ti;
        tj = int(u) - ti * (ti + 1) / 2;
    } else {  // bands of four tiles' rows: what an XCD works on at a time is nearly square
        const int band = int(u) / (4 * nj), in = int(u) - band * 4 * nj, high = min(4, ni - 4 * band);
        tj = in / high;
        ti = 4 * band + in - tj * high;
    }
    ti = __builtin_amdgcn_readfirstlane(ti);
    tj = __builtin_amdgcn_readfirstlane(tj);
    const int K = kPair * (MODE == kGram ? t.cp : t.rp);  // numbers of I's rows
    const _Float16* X = t.x[s.from] + kPair * int64_t(which) * t.rp * t.cp;
    const _Float16* A = t.a + kPair * int64_t(which) * t.rp * t.rp;
    const _Float16* B = t.b + kPair * int64_t(which) * t.rp * t.rp;
    const _Float16* I = (MODE == kGram ? X : MODE == kPoly ? A : B) + int64_t(ti) * BT * K;
    const _Float16* J = TR ? X + kPair * tj * BT : (MODE == kGram ? X : A) + int64_t(tj) * BT * K;

    const RowPlace in = row_place();
    const uint32_t irow = 2 * (uint32_t(in.row) * K + in.number);  // bytes
    const int64_t istep = int64_t(32) * K, jld = kPair * int64_t(t.cp);
    uint32_t jrow[TR ? FETCH : 1];
    if constexpr (TR) {
#pragma unroll
        for (int n = 0; n < FETCH; ++n) {
            const SumPlace at_n = sum_place<BT, kPair>(n);
            jrow[n] = 2 * (uint32_t(at_n.sum) * uint32_t(jld) + at_n.number);
        }
    }
    auto load = [&](int c, int n, short* to) {
        if (n < FETCH) load_lds(I + c * kRow + n * istep, irow, to);
        else if constexpr (TR) load_lds(J + c * (kRow / kPair) * jld, jrow[n - FETCH], to);
        else load_lds(J + c * kRow + (n - FETCH) * istep, irow, to);
    };
    Acc<BT> acc;
    clear<BT>(acc);
    products<BT, kPair, false, TR, false>(lds, K / kRow, acc, load, [](int) {});  // sides are multiples of 128

    // The result, 32 rows of a wavefront's part at a time by way of LDS (its own part of it), from where rows and, for the
    // second place of a symmetric one and for tall matrices' parameters, columns leave 8 values a lane.  acc[m][n][q] is
    // of row 32 m + l32 and column 32 n + 8 (q / 4) + 4 half + q % 4.
    float own = s.own, prod = s.prod;
    if (s.first) {
        const float rho = stats[t.stat0 + which].rho;
        if (MODE == kGram) prod *= rho * rho;
        if (MODE == kUpdate || MODE == kFinal) {
            own *= rho;
            prod *= rho;
        }
    }
    const int width = SYM ? t.rp : t.cp;
    const int64_t ld = kPair * int64_t(width);
    const _Float16* E = MODE == kPoly ? A : X;
    _Float16* out = (MODE == kGram ? t.a : MODE == kPoly ? t.b : t.x[s.from ^ 1]) + int64_t(which) * t.rp * ld;
    float decay = 0, rate = -ap.inv;  // of p and of its change; the result itself has no p
    if (MODE == kFinal && t.m) {
        const float lr = ap.lr_device ? *ap.lr_device : ap.lr;
        decay = 1 - lr * ap.wd;
        rate = lr * t.adjust * ap.inv;
    }
    const bool tall = t.rows > t.cols;
    const int64_t off = int64_t(which) * t.rows * t.cols;
    // Symmetric results are stored from the diagonal downwards and from there above it, on the diagonal's own 32 x 32 blocks
    // too: the two halves' sums run in different orders with pairs, and results would differ with the size of tiles.
    const bool columns = SYM || (MODE == kFinal && tall), corner = SYM && ti == tj && wi == wj;
    constexpr int LD = W + 4, ITEMS = W / 16;  // items of 8 values a lane
    float* part = reinterpret_cast<float*>(lds + wave * 2 * 32 * LD);
    const int j0 = tj * BT + wj * W;
    __syncthreads();
    if (SYM && ti == tj && wi < wj) return;  // above the diagonal
    // What a strip reads of E is loaded while the one before it leaves, where there are registers for both
    constexpr bool EARLY = MODE != kGram && BT <= 128;
    half8 old[EARLY ? 2 : 1][MODE == kGram ? 1 : kPair][ITEMS];
    auto load_old = [&](int m, auto& to) {
#pragma unroll
        for (int it = 0; it < ITEMS; ++it) {
            const int item = it * 64 + lane;
            const int i = min(ti * BT + wi * W + 32 * m + item / (W / 8), t.rp - 1), j = min(j0 + item % (W / 8) * 8, width - 8);
#pragma unroll
            for (int pl = 0; pl < kPair; ++pl)
                to[pl][it] = *reinterpret_cast<const half8*>(E + int64_t(i) * ld + place(j) + 16 * pl);
        }
    };
    if constexpr (EARLY) load_old(0, old[0]);
    auto strip = [&](auto type, auto at_m) {
        constexpr int m = decltype(at_m)::value, now = EARLY ? m & 1 : 0;
        using P = decltype(type);
        P* const p = static_cast<P*>(t.p) + off;
        const int i0 = ti * BT + wi * W + 32 * m;
        if constexpr (MODE != kGram && !EARLY) load_old(m, old[0]);
        typename Eight<P>::V par[MODE == kFinal ? ITEMS : 1];
        if constexpr (MODE == kFinal) {
#pragma unroll
            for (int it = 0; it < ITEMS; ++it) {
                const int item = it * 64 + lane;
                const int i = i0 + (tall ? item % 4 * 8 : item / (W / 8)), j = j0 + (tall ? item / 4 : item % (W / 8) * 8);
                const bool whole = tall ? i + 8 <= t.r && j < t.c : i < t.r && j + 8 <= t.c;
                if (whole && decay != 0)
                    par[it] = *reinterpret_cast<const typename Eight<P>::V*>(
                        p + (tall ? int64_t(j) * t.cols + i : int64_t(i) * t.cols + j));
            }
        }
#pragma unroll
        for (int n = 0; n < MT; ++n)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = prod * acc[m][n][4 * q + e];
                *reinterpret_cast<f32x4*>(part + l32 * LD + 32 * n + 8 * q + 4 * half) = v;
            }
        if constexpr (EARLY && m + 1 < MT) load_old(m + 1, old[(m + 1) & 1]);
        wave_sync();
#pragma unroll
        for (int it = 0; it < ITEMS; ++it) {
            const int item = it * 64 + lane, r = item / (W / 8), i = i0 + r, jj = item % (W / 8) * 8, j = j0 + jj;
            const int block = corner ? (jj >> 5) - m : -1;  // 0: the diagonal's; above it, nothing is stored
            if (i >= t.rp || j >= width || block > 0) continue;
            float v[8];
            if (block < 0) {
                *reinterpret_cast<f32x4*>(v) = *reinterpret_cast<const f32x4*>(part + r * LD + jj);
                *reinterpret_cast<f32x4*>(v + 4) = *reinterpret_cast<const f32x4*>(part + r * LD + jj + 4);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int c = jj + e - 32 * m;
                    v[e] = part[max(r, c) * LD + 32 * m + min(r, c)];
                }
            }
            if constexpr (MODE != kGram) {
#pragma unroll
                for (int pl = kPair - 1; pl >= 0; --pl)
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] += own * float(old[now][pl][it][e]);
                if (columns && block < 0) {
                    *reinterpret_cast<f32x4*>(part + r * LD + jj) = *reinterpret_cast<const f32x4*>(v);
                    *reinterpret_cast<f32x4*>(part + r * LD + jj + 4) = *reinterpret_cast<const f32x4*>(v + 4);
                }
            }
            if constexpr (MODE == kFinal) {
                if (!tall && i < t.r) apply(p + int64_t(i) * t.cols + j, t.c - j, par[it], decay, rate, v);
            } else {
                put8(out + int64_t(i) * ld + place(j), v);
            }
        }
        wave_sync();
        if (columns) {
#pragma unroll
            for (int it = 0; it < ITEMS; ++it) {
                const int item = it * 64 + lane, jj = item / 4, j = j0 + jj, r = item % 4 * 8, i = i0 + r;
                if (i >= t.rp || j >= width || (corner && (jj >> 5) >= m)) continue;
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = part[(r + e) * LD + jj];
                if constexpr (MODE == kFinal) {
                    if (j < t.c) apply(p + int64_t(j) * t.cols + i, t.r - i, par[it], decay, rate, v);
                } else {
                    put8(out + int64_t(j) * ld + place(i), v);
                }
            }
            wave_sync();
        }
    };
    auto strips = [&](auto type) {
        strip(type, std::integral_constant<int, 0>());
        if constexpr (MT > 1) strip(type, std::integral_constant<int, 1>());
        if constexpr (MT > 2) strip(type, std::integral_constant<int, 2>());
        if constexpr (MT > 3) strip(type, std::integral_constant<int, 3>());
    };
    if constexpr (MODE != kFinal) strips(float{});  // the type is of the parameters
    else by_type(t.dtype, strips);
}

// ---------------------------------------------------------------------------
// Small matrices
// ---------------------------------------------------------------------------

// Rows of a small matrix in LDS: 48 bytes more than their values, so that 16 rows' pieces of 16 bytes meet every bank once.
inline __host__ __device__ int small_row(int cols) { return 2 * cols + 48; }

// Bytes that X and A of an r x c matrix take there.
inline int64_t small_bytes(int64_t r, int64_t c) {
    const int64_t rq = ceil_div(r, 32) * 32, cq = ceil_div(c, 32) * 32;
    return kPair * rq * (small_row(int(rq)) + 2 * cq + 48);
}

constexpr int kSmallThreads = 512, kSmallSide = 128;  // the smaller side's limit: four blocks of 32 rows
constexpr int kSmallLds[] = {48 << 10, (160 << 10) - 512};

// The factors of every step.
struct Steps {
    float gram[MNX_MUON_MAX_STEPS], poly_own[MNX_MUON_MAX_STEPS], poly[MNX_MUON_MAX_STEPS], own[MNX_MUON_MAX_STEPS],
        prod[MNX_MUON_MAX_STEPS];
    int count;
};

// What k_muon_small reads of a tensor.  Up to 32 of them travel in its arguments, and the launch that writes the table is
// not needed (64 x 64 float32: 30 us, 33 with it).
struct SmallMat {
    void* p;
    const void* g;
    float* m;
    int32_t rows, cols, dtype;
    float adjust;
    uint32_t stat0;
};
constexpr int kSmallArgs = 32;
struct SmallList {
    SmallMat mat[kSmallArgs];
};
static_assert(sizeof(SmallList) + sizeof(Steps) <= 3840, "4 KB of arguments");

// A whole matrix in one workgroup, from its gradient to its parameters: X and A (then B) stay in LDS, and one launch does
// what takes 19 with tiles.  One matrix of 128 x 128 takes 61 us so and 74 with tiles, 64 x 64 30 and 74; 300 of 128 x 128
// 123 and 269.  It is bound by latency: about 11 us a step at 128 x 128, products that depend on the last ones with two
// wavefronts a SIMD.
//
// Eight wavefronts share the blocks of 32 x 32 of A and B on and below the diagonal, and the columns of X, 32 at a time:
// such columns of a X + B X read nothing of X but these columns, so they are replaced in place.  Sums of hi hi and of the
// cross products run apart, and are added at the end.
template <int LDS, bool ARGS>
__global__ void __launch_bounds__(kSmallThreads) k_muon_small(SmallList list, const Mat* __restrict__ table, int count,
                                                              Momentum h, double eps, Steps st, Apply ap) {
    __shared__ __attribute__((aligned(16))) char lds[LDS];
    __shared__ double part[kSmallThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    constexpr int WAVES = kSmallThreads / 64;
    SmallMat t;
    if constexpr (ARGS) {
        const bool mine = lane < count && list.mat[min(lane, kSmallArgs - 1)].stat0 <= blockIdx.x;
        t = list.mat[__builtin_amdgcn_readfirstlane(__popcll(__ballot(mine)) - 1)];
    } else {
        const Mat& m = table[find_mat(table, count, &Mat::stat0, blockIdx.x)];
        t = {m.p, m.g, m.m, m.rows, m.cols, m.dtype, m.adjust, m.stat0};
    }
    const int64_t n = int64_t(t.rows) * t.cols, off = int64_t(blockIdx.x - t.stat0) * n;
    const bool tall = t.rows > t.cols;
    const int tr = min(t.rows, t.cols), tc = max(t.rows, t.cols);
    const int rb = (tr + 31) / 32, cb = (tc + 31) / 32;  // blocks of 32
    const int sx = small_row(32 * cb), sa = small_row(32 * rb);
    char* const X = lds;
    char* const A = lds + kPair * 32 * rb * sx;
    const int xplane = 32 * rb * sx, aplane = 32 * rb * sa;

    // momenta and the norm, four vectors a thread on their way at a time
    double sum = 0;
    by_type(t.dtype, [&](auto type) {
        const auto* g = static_cast<const decltype(type)*>(t.g) + off;
        for (int64_t i0 = tid * 4; i0 < n; i0 += kSmallThreads * 16) {
            float v[4][4], m[4][4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int64_t i = i0 + k * kSmallThreads * 4;
                load4(g + i, n - i, v[k]);
                if (t.m) load4(t.m + off + i, n - i, m[k]);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int64_t i = i0 + k * kSmallThreads * 4;
                if (t.m) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (h.maximize) v[k][e] = -v[k][e];
                        m[k][e] = __builtin_fmaf(h.mu, m[k][e], h.w * v[k][e]);
                        v[k][e] = direction(v[k][e], m[k][e], h);
                    }
                    store4(t.m + off + i, n - i, m[k]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) sum += double(v[k][e]) * double(v[k][e]);
            }
        }
    });
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if (lane == 0) part[wave] = sum;
    __syncthreads();
    sum = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) sum += part[w];
    const Stat stat = stat_of(sqrt(sum), eps);

    // X: u by its own rows, four of their values a thread
    by_type(t.dtype, [&](auto type) {
        const auto* g = static_cast<const decltype(type)*>(t.g) + off;
        const int rows = 32 * (tall ? cb : rb), vecs = 8 * (tall ? rb : cb);
        for (int it0 = tid; it0 < rows * vecs; it0 += 4 * kSmallThreads) {
            float v[4][4], m[4][4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int it = it0 + k * kSmallThreads, i = it / vecs, j = it % vecs * 4;
                const int left = i < t.rows ? t.cols - j : 0;
                load4(g + int64_t(i) * t.cols + j, left, v[k]);
                if (t.m) load4(t.m + off + int64_t(i) * t.cols + j, left, m[k]);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int it = it0 + k * kSmallThreads, i = it / vecs, j = it % vecs * 4;
                if (it >= rows * vecs) continue;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (t.m) v[k][e] = direction(h.maximize ? -v[k][e] : v[k][e], m[k][e], h);
                    v[k][e] = ldexpf(v[k][e], stat.exponent);
                }
                if (!tall) {
                    put4(reinterpret_cast<_Float16*>(X + i * sx + 2 * j), xplane / 2, v[k]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        _Float16* to = reinterpret_cast<_Float16*>(X + (j + e) * sx + 2 * i);
                        to[0] = _Float16(v[k][e]);
                        to[xplane / 2] = _Float16(v[k][e] - float(to[0]));
                    }
                }
            }
        }
    });
    __syncthreads();

    auto rows_of = [&](const char* base, int stride, int block, int k) {
        return *reinterpret_cast<const half8*>(base + (32 * block + l32) * stride + 2 * (k + 8 * half));
    };
    auto cols_of = [&](const char* base, int stride, int block, int k) {
        const char* q = base + (k + 8 * half + ((lane & 15) >> 2)) * stride + 2 * (32 * block + (l32 & 16) + (lane & 3) * 4);
        return __builtin_bit_cast(half8, read_tr(q, q + 4 * stride));
    };
    auto zero = [] {
        f32x16 z;
#pragma unroll
        for (int q = 0; q < 16; ++q) z[q] = 0.f;
        return z;
    };
    // block (bi, bj) of the product of S's rows with themselves
    auto square = [&](const char* S, int stride, int plane, int bi, int bj, int K) {
        f32x16 big = zero(), low = zero(), high = zero();
#pragma unroll 4
        for (int k = 0; k < K; k += 16) {
            const half8 i = rows_of(S, stride, bi, k), j = rows_of(S, stride, bj, k);
            const half8 il = rows_of(S + plane, stride, bi, k), jl = rows_of(S + plane, stride, bj, k);
            low = mfma(jl, i, low);
            high = mfma(j, il, high);
            big = mfma(j, i, big);
        }
        return big + (low + high);
    };
    // the block's values into A, above the diagonal too; `own` of what is there
    auto into_a = [&](const f32x16& acc, int bi, int bj, float own, float prod) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int i = 32 * bi + l32, j = 32 * bj + 8 * q + 4 * half;
            _Float16* to = reinterpret_cast<_Float16*>(A + i * sa + 2 * j);
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = prod * acc[4 * q + e];
            if (own != 0) {
#pragma unroll
                for (int pl = kPair - 1; pl >= 0; --pl) {
                    const half4 old = *reinterpret_cast<const half4*>(to + pl * (aplane / 2));
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] += own * float(old[e]);
                }
            }
            put4(to, aplane / 2, v);
            if (bi != bj) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    _Float16* mirror = reinterpret_cast<_Float16*>(A + (j + e) * sa + 2 * i);
                    const _Float16 hi = _Float16(v[e]);
                    mirror[0] = hi;
                    mirror[aplane / 2] = _Float16(v[e] - float(hi));
                }
            }
        }
    };
    auto block_of = [](int b, int& bi, int& bj) {  // the b-th on and below the diagonal
        bi = b >= 6 ? 3 : b >= 3 ? 2 : b >= 1 ? 1 : 0;
        bj = b - bi * (bi + 1) / 2;
    };
    const int blocks = rb * (rb + 1) / 2;
    float decay = 0, rate = -ap.inv;
    if (t.m) {
        const float lr = ap.lr_device ? *ap.lr_device : ap.lr;
        decay = 1 - lr * ap.wd;
        rate = lr * t.adjust * ap.inv;
    }
#pragma unroll 1
    for (int step = 0; step < st.count; ++step) {
        const float rho = step == 0 ? stat.rho : 1.f;
        for (int b = wave; b < blocks; b += WAVES) {
            int bi, bj;
            block_of(b, bi, bj);
            into_a(square(X, sx, xplane, bi, bj, 32 * cb), bi, bj, 0.f, st.gram[step] * rho * rho);
        }
        __syncthreads();
        {
            int bi[2], bj[2];
            f32x16 acc[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int b = wave + k * WAVES;
                if (b < blocks) {
                    block_of(b, bi[k], bj[k]);
                    acc[k] = square(A, sa, aplane, bi[k], bj[k], 32 * rb);
                }
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < 2; ++k)
                if (wave + k * WAVES < blocks) into_a(acc[k], bi[k], bj[k], st.poly_own[step], st.poly[step]);
        }
        __syncthreads();
        const float own = st.own[step] * rho, prod = st.prod[step] * rho;
        const bool last = step + 1 == st.count;
        // with more than two blocks of rows, two wavefronts share 32 columns, and wait for each other before they replace them
        const int groups = (rb + 1) / 2;
        for (int item0 = 0; item0 < cb * groups; item0 += WAVES) {
            const int item = item0 + wave, bj = item / groups, r0 = item % groups * 2;
            const bool mine = item < cb * groups;
            f32x16 big[2], small[2];
            if (mine) {
#pragma unroll
                for (int r = 0; r < 2; ++r) big[r] = small[r] = zero();
#pragma unroll 2
                for (int k = 0; k < 32 * rb; k += 16) {
                    const half8 j = cols_of(X, sx, bj, k);
                    half8 i[2], il[2];
#pragma unroll
                    for (int r = 0; r < 2; ++r) i[r] = rows_of(A, sa, min(r0 + r, rb - 1), k);
                    const half8 jl = cols_of(X + xplane, sx, bj, k);
#pragma unroll
                    for (int r = 0; r < 2; ++r) il[r] = rows_of(A + aplane, sa, min(r0 + r, rb - 1), k);
#pragma unroll
                    for (int r = 0; r < 2; ++r) small[r] = mfma(jl, i[r], small[r]);
#pragma unroll
                    for (int r = 0; r < 2; ++r) big[r] = mfma(j, i[r], big[r]);
#pragma unroll
                    for (int r = 0; r < 2; ++r) small[r] = mfma(j, il[r], small[r]);
                }
            }
            if (groups > 1) __syncthreads();
            else wave_sync();
            if (!mine) continue;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                if (r0 + r >= rb) continue;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int i = 32 * (r0 + r) + l32, j = 32 * bj + 8 * q + 4 * half;
                    _Float16* to = reinterpret_cast<_Float16*>(X + i * sx + 2 * j);
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        v[e] = prod * (big[r][4 * q + e] + small[r][4 * q + e]);
#pragma unroll
                    for (int pl = kPair - 1; pl >= 0; --pl) {
                        const half4 old = *reinterpret_cast<const half4*>(to + pl * (xplane / 2));
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] += own * float(old[e]);
                    }
                    put4(to, xplane / 2, v);
                    if (!last || i >= tr) continue;
                    by_type(t.dtype, [&](auto type) {
                        auto* p = static_cast<decltype(type)*>(t.p) + off;
                        const int step_ = tall ? t.cols : 1;
                        auto* to_p = p + (tall ? int64_t(j) * t.cols + i : int64_t(i) * t.cols + j);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (j + e < tc) {
                                auto& par = to_p[int64_t(e) * step_];
                                par = decltype(type)(stepped(decay != 0 ? decay * float(par) : 0.f, v[e], rate));
                            }
                    });
                }
            }
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

struct Scales {
    std::vector<double> x;  // of X before each step and after the last
    std::vector<double> a, b;
};

// Bounds of what the iteration can reach from singular values in [0, 1], as powers of two; false where it diverges.
bool bounds(const mnx_muon_args& args, Scales& s) {
    const double a = args.coefficients[0], b = args.coefficients[1], c = args.coefficients[2];
    auto scale = [](double bound) { return std::ldexp(1.0, 12 - int(std::ceil(std::log2(std::max(bound, 1.0) / 4)))); };
    double n = 1.02;  // roundings included
    for (int k = 0; k < args.steps; ++k) {
        const double l = n * n;
        double top_b = std::fabs(b * l + c * l * l), top_x = std::fabs(a * n + b * n * l + c * n * l * l);
        if (c != 0) {
            const double v = -b / (2 * c);
            if (v > 0 && v < l) top_b = std::max(top_b, std::fabs(b * v + c * v * v));
            const double disc = 9 * b * b - 20 * a * c;
            for (int sign = -1; disc >= 0 && sign <= 1; sign += 2) {
                const double z = (-3 * b + sign * std::sqrt(disc)) / (10 * c);
                if (z > 0 && z < l)
                    top_x = std::max(top_x, std::sqrt(z) * std::fabs(a + b * z + c * z * z));
            }
        } else if (b != 0) {
            const double z = -a / (3 * b);
            if (z > 0 && z < l) top_x = std::max(top_x, std::sqrt(z) * std::fabs(a + b * z));
        }
        s.x.push_back(scale(n));
        s.a.push_back(scale(l));
        s.b.push_back(scale(top_b));
        n = 1.02 * top_x;
        if (!(n < 64) || !(top_b < 4096)) return false;
    }
    s.x.push_back(scale(n));
    return true;
}

struct Plan {
    std::vector<Mat> mat;
    Prefix total{};
    uint32_t stats = 0;
    size_t bytes = 0;
    int sym_tile = 128, upd_tile = 128;
    int64_t lds = 0;
    double* partial = nullptr;
    Stat* stat = nullptr;
    Mat* table = nullptr;
};

inline int64_t up(int64_t n, int64_t m) { return ceil_div(n, m) * m; }

int check_args(const mnx_muon_args& a) {
    MNX_REQUIRE(a.count >= 0 && (a.count == 0 || (a.batch && a.rows && a.cols && a.dtype)), "muon: null pointer");
    MNX_REQUIRE(a.steps >= 1 && a.steps <= MNX_MUON_MAX_STEPS, "muon: 1 to %d steps, got %d", MNX_MUON_MAX_STEPS, a.steps);
    MNX_REQUIRE(a.eps >= 0 && a.eps < HUGE_VAL, "muon: eps %g", a.eps);
    for (double v : a.coefficients) MNX_REQUIRE(std::isfinite(v), "muon: coefficients must be finite");
    for (int64_t i = 0; i < a.count; ++i) {
        MNX_REQUIRE(a.batch[i] >= 0 && a.rows[i] >= 0 && a.cols[i] >= 0 && a.rows[i] <= MNX_MUON_MAX_SIDE &&
                        a.cols[i] <= MNX_MUON_MAX_SIDE,
                    "muon: tensor %lld has %lld matrices of %lld x %lld; sides are at most %d", (long long)i,
                    (long long)a.batch[i], (long long)a.rows[i], (long long)a.cols[i], MNX_MUON_MAX_SIDE);
        MNX_REQUIRE(elem_valid(a.dtype[i]), "muon: tensor %lld has an unknown type", (long long)i);
    }
    return MNX_OK;
}

// Tiles of a tensor's symmetric products, or of its updates.
inline int64_t tiles_of(const Mat& t, bool sym, int tile) {
    const int64_t ni = ceil_div(t.rp, tile), nj = ceil_div(t.cp, tile);
    return t.batch * (sym ? ni * (ni + 1) / 2 : ni * nj);
}

constexpr int kTile[] = {256, 192, 128, 64}, kTiles = 4;

// The time of a launch, about, in microseconds, by which the size of its tiles is chosen (64 matrices of 512 x 512: 256; one
// of 4096 x 4096: 192 for A and B, 256 for B X; one of 2048 x 2048: 64 and 128; one of 1024 x 1024: 64).  A tile's begin and
// end take 4, a chunk of 64 single numbers 1.95 (256), 1.1 (192) or 0.23 (64), with one tile a CU; tiles of 128 share a CU
// two by two, 1.05 a chunk, or 0.6 where they are few; 32 pairs half as much again (a third product; tiles of 64 wait for
// memory).  `mats` are sorted: the longest tiles start first, each on the CU that is free first.
double cost(const std::vector<Mat>& mats, int kind, int tile) {
    double tiles = 0;
    for (const Mat& t : mats) tiles += double(tiles_of(t, kind != kUpdate, tile));
    const bool two = tile == 128 && tiles > 256;
    const double slots = two ? 512 : 256;
    double chunk = tile == 256 ? 1.95 : tile == 192 ? 1.1 : two ? 1.05 : tile == 128 ? 0.6 : 0.23;
    if (tile != 64) chunk *= 1.5;
    auto one = [&](const Mat& t) { return 4 + chunk * kPair * double(kind == kGram ? t.cp : t.rp) / kRow; };
    if (tiles > 16 * slots) {  // many rounds: their sum
        double all = 0;
        for (const Mat& t : mats) all += one(t) * double(tiles_of(t, kind != kUpdate, tile));
        return all / slots;
    }
    std::vector<std::pair<double, double>> free{{0.0, slots}};  // when so many slots are free
    for (size_t i = 0; i < mats.size();) {
        const double time = one(mats[i]);
        double n = 0;
        for (; i < mats.size() && one(mats[i]) == time; ++i) n += double(tiles_of(mats[i], kind != kUpdate, tile));
        while (n > 0) {
            auto at = std::min_element(free.begin(), free.end());
            const double begin = at->first, some = std::min(n, at->second);
            n -= some;
            if ((at->second -= some) == 0) free.erase(at);
            const double end = begin + time;
            auto same = std::find_if(free.begin(), free.end(), [&](const auto& f) { return f.first == end; });
            if (same != free.end()) same->second += some;
            else free.emplace_back(end, some);
        }
    }
    return std::max_element(free.begin(), free.end())->first;
}

// Whether one workgroup takes a whole matrix (at most LDS holds: 128 x 128 or 64 x 512).  300 matrices of 32 x 256 take
// 59 us so and 298 with tiles.
inline bool is_small(int64_t rows, int64_t cols) {
    return std::min(rows, cols) <= kSmallSide && std::max(rows, cols) <= 4096 &&
           small_bytes(std::min(rows, cols), std::max(rows, cols)) <= kSmallLds[1];
}

// Lays the tensors of small matrices, or the others, out over the workspace (from `base`, which may be null for its size
// alone).
int lay_out(const mnx_muon_args& a, bool small, char* base, Plan& plan) {
    Workspace ws{base, 0};
    uint64_t chunk = 0, cast = 0, stat = 0;
    std::vector<int64_t> order(size_t(a.count));  // the largest first: their tiles take longest
    std::iota(order.begin(), order.end(), int64_t(0));
    std::stable_sort(order.begin(), order.end(), [&](int64_t i, int64_t j) {
        const int64_t x = std::min(a.rows[i], a.cols[i]), y = std::min(a.rows[j], a.cols[j]);
        return x != y ? x > y : std::max(a.rows[i], a.cols[i]) > std::max(a.rows[j], a.cols[j]);
    });
    for (const int64_t i : order) {
        if (!a.batch[i] || !a.rows[i] || !a.cols[i] || is_small(a.rows[i], a.cols[i]) != small) continue;
        Mat t{};
        t.rows = int32_t(a.rows[i]);
        t.cols = int32_t(a.cols[i]);
        t.r = std::min(t.rows, t.cols);
        t.c = std::max(t.rows, t.cols);
        t.rp = int32_t(up(t.r, kPad));
        t.cp = int32_t(up(t.c, kPad));
        t.batch = int32_t(a.batch[i]);
        t.dtype = a.dtype[i];
        t.p = a.params ? a.params[i] : nullptr;
        t.g = a.grads ? a.grads[i] : nullptr;
        t.m = a.momenta ? a.momenta[i] : nullptr;
        t.adjust = a.adjust == 0 ? float(std::sqrt(std::max(1.0, double(t.rows) / t.cols)))
                                 : float(0.2 * std::sqrt(double(t.c)));
        t.stat0 = uint32_t(stat);
        t.chunk0 = uint32_t(chunk);
        t.cast0 = uint32_t(cast);
        const uint64_t b = uint64_t(a.batch[i]);
        stat += b;
        MNX_REQUIRE(std::max(b, stat) < (1u << 22), "muon: too many matrices in one call");
        if (small) {
            plan.lds = std::max(plan.lds, small_bytes(t.r, t.c));
            plan.mat.push_back(t);
            continue;
        }
        chunk += b * uint64_t(ceil_div(int64_t(t.rows) * t.cols, kChunk));
        cast += b * uint64_t(t.rp / kCast) * (t.cp / kCast);
        for (_Float16*& x : t.x) x = ws.take<_Float16>(size_t(kPair * a.batch[i] * t.rp * t.cp));
        t.a = ws.take<_Float16>(size_t(kPair * a.batch[i] * t.rp * t.rp));
        t.b = ws.take<_Float16>(size_t(kPair * a.batch[i] * t.rp * t.rp));
        // a grid has fewer than 2^32 threads
        MNX_REQUIRE(std::max(chunk, cast) < (1u << 23), "muon: too many matrices in one call");
        plan.mat.push_back(t);
    }
    if (small) {
        plan.stats = uint32_t(stat);
        plan.table = ws.take<Mat>(plan.mat.size());
        plan.bytes = ws.used;
        return MNX_OK;
    }
    for (int kind : {kGram, kUpdate}) {
        int best = 0;
        double least = HUGE_VAL;
        for (int k = 0; k < kTiles; ++k) {
            const double c = cost(plan.mat, kind, kTile[k]);
            if (c < least) {
                least = c;
                best = k;
            }
        }
        (kind == kGram ? plan.sym_tile : plan.upd_tile) = kTile[best];
    }
    uint64_t sym = 0, upd = 0;
    for (Mat& t : plan.mat) {
        t.sym0 = uint32_t(sym);
        t.upd0 = uint32_t(upd);
        sym += uint64_t(tiles_of(t, true, plan.sym_tile));
        upd += uint64_t(tiles_of(t, false, plan.upd_tile));
    }
    MNX_REQUIRE(std::max(sym, upd) < (1u << 23), "muon: too many matrices in one call");
    plan.total = {uint32_t(chunk), uint32_t(cast), uint32_t(sym), uint32_t(upd)};
    // the last tiles read past the last matrix
    int64_t past = 0;
    for (const Mat& t : plan.mat) past = std::max<int64_t>(past, int64_t(256) * kPair * t.cp);
    if (past) ws.take<_Float16>(size_t(past));
    plan.stats = uint32_t(stat);
    plan.partial = ws.take<double>(size_t(chunk));
    plan.stat = ws.take<Stat>(size_t(stat));
    plan.table = ws.take<Mat>(plan.mat.size());
    plan.bytes = ws.used;
    return MNX_OK;
}

template <int MODE>
int product(const Plan& plan, const Step& s, const Apply& ap, mnx_stream_t stream) {
    constexpr bool SYM = MODE == kGram || MODE == kPoly;
    const int tile = SYM ? plan.sym_tile : plan.upd_tile;
    const uint32_t units = SYM ? plan.total.sym : plan.total.upd, grid = uint32_t(up(units, 128));
    const int count = int(plan.mat.size());
    const auto kernel = tile == 256 ? k_muon_product<MODE, 256>
                        : tile == 192 ? k_muon_product<MODE, 192>
                        : tile == 128 ? k_muon_product<MODE, 128> : k_muon_product<MODE, 64>;
    kernel<<<grid, 256, 0, stream>>>(plan.table, count, units, s, plan.stat, ap);
    MNX_CHECK_LAUNCH();
    return MNX_OK;
}

int write_table(const Plan& plan, mnx_stream_t stream) {
    const int count = int(plan.mat.size());
    for (int at = 0; at < count; at += kTableArgs) {
        TableArgs t;
        t.first = at;
        t.count = std::min(kTableArgs, count - at);
        for (int i = 0; i < t.count; ++i) t.mat[i] = plan.mat[size_t(at + i)];
        k_muon_table<<<1, 256, 0, stream>>>(t, plan.table);
        MNX_CHECK_LAUNCH();
    }
    return MNX_OK;
}

// The factors of step k's three products.
struct Factors {
    Step gram, poly, update;
};
Factors factors(const mnx_muon_args& a, const Scales& sc, int k) {
    const double ca = a.coefficients[0], cb = a.coefficients[1], cc = a.coefficients[2];
    const double A = sc.a[size_t(k)], B = sc.b[size_t(k)];
    const int from = k & 1, first = k == 0;
    const double xs = first ? 4096.0 : sc.x[size_t(k)];  // the first X is stored at 2^12 whatever the bounds say
    const double to = k + 1 == a.steps ? 1.0 : sc.x[size_t(k) + 1];
    return {{0.f, float(A / (xs * xs)), from, first},
            {float(B * cb / A), float(B * cc / (A * A)), from, first},
            {float(to * ca / xs), float(to / (B * xs)), from, first}};
}

int run(const mnx_muon_args& a, const Plan& plan, const Scales& sc, mnx_stream_t stream) {
    const int count = int(plan.mat.size());
    if (!count) return MNX_OK;
    if (int rc = write_table(plan, stream)) return rc;
    const Momentum h{float(a.momentum), float(1 - a.momentum), a.nesterov, a.maximize};
    k_muon_momentum<<<plan.total.chunk, 256, 0, stream>>>(plan.table, count, h, plan.partial);
    MNX_CHECK_LAUNCH();
    k_muon_norm<<<plan.stats, 256, 0, stream>>>(plan.table, count, plan.partial, a.eps, plan.stat);
    MNX_CHECK_LAUNCH();
    k_muon_cast<<<plan.total.cast, 256, 0, stream>>>(plan.table, count, h, plan.stat);
    MNX_CHECK_LAUNCH();
    const Apply none{}, ap{float(a.lr), a.lr_device, float(a.weight_decay), 1.0f};
    for (int k = 0; k < a.steps; ++k) {
        const Factors f = factors(a, sc, k);
        if (int rc = product<kGram>(plan, f.gram, none, stream)) return rc;
        if (int rc = product<kPoly>(plan, f.poly, none, stream)) return rc;
        if (int rc = k + 1 == a.steps ? product<kFinal>(plan, f.update, ap, stream)
                                      : product<kUpdate>(plan, f.update, none, stream))
            return rc;
    }
    return MNX_OK;
}

int run_small(const mnx_muon_args& a, const Plan& plan, const Scales& sc, mnx_stream_t stream) {
    const int count = int(plan.mat.size());
    if (!count) return MNX_OK;
    SmallList list{};
    const bool args = count <= kSmallArgs;
    if (args) {
        for (int i = 0; i < count; ++i) {
            const Mat& m = plan.mat[size_t(i)];
            list.mat[i] = {m.p, m.g, m.m, m.rows, m.cols, m.dtype, m.adjust, m.stat0};
        }
    } else if (int rc = write_table(plan, stream)) {
        return rc;
    }
    const Momentum h{float(a.momentum), float(1 - a.momentum), a.nesterov, a.maximize};
    const Apply ap{float(a.lr), a.lr_device, float(a.weight_decay), 1.0f};
    Steps st;
    st.count = a.steps;
    for (int k = 0; k < a.steps; ++k) {
        const Factors f = factors(a, sc, k);
        st.gram[k] = f.gram.prod;
        st.poly_own[k] = f.poly.own;
        st.poly[k] = f.poly.prod;
        st.own[k] = f.update.own;
        st.prod[k] = f.update.prod;
    }
    const auto kernel = plan.lds <= kSmallLds[0] ? (args ? k_muon_small<kSmallLds[0], true> : k_muon_small<kSmallLds[0], false>)
                                                 : (args ? k_muon_small<kSmallLds[1], true> : k_muon_small<kSmallLds[1], false>);
    kernel<<<plan.stats, kSmallThreads, 0, stream>>>(list, plan.table, count, h, a.eps, st, ap);
    MNX_CHECK_LAUNCH();
    return MNX_OK;
}

// The tensors of a call by how they are multiplied: each kind's launches follow the last one's, in the same workspace.
struct Form {
    bool small;
    int (*run)(const mnx_muon_args&, const Plan&, const Scales&, mnx_stream_t);
};
constexpr Form kForms[] = {{true, run_small}, {false, run}};

}  // namespace
}  // namespace mnx

using namespace mnx;

extern "C" {

size_t mnx_muon_workspace_bytes(const mnx_muon_args* args) {
    clear_error();
    if (!args || check_args(*args) != MNX_OK) return 0;
    size_t most = 256;
    for (const Form& f : kForms) {
        Plan plan;
        if (lay_out(*args, f.small, nullptr, plan) != MNX_OK) return 0;
        most = std::max(most, plan.bytes);
    }
    return most;
}

int mnx_muon_step(const mnx_muon_args* args, mnx_stream_t stream) {
    clear_error();
    MNX_REQUIRE(args, "muon: null arguments");
    const mnx_muon_args& a = *args;
    if (int rc = check_args(a)) return rc;
    MNX_REQUIRE(a.momentum >= 0 && a.momentum < 1, "muon: 0 <= momentum < 1, got %g", a.momentum);
    MNX_REQUIRE(a.adjust == 0 || a.adjust == 1, "muon: adjust 0 or 1, got %d", a.adjust);
    MNX_REQUIRE(a.count == 0 || (a.params && a.grads), "muon: null pointer");
    for (int64_t i = 0; i < a.count; ++i)
        MNX_REQUIRE(!a.batch[i] || !a.rows[i] || !a.cols[i] ||
                        (a.params[i] && a.grads[i] && (!a.momenta || a.momenta[i])),
                    "muon: tensor %lld has a null pointer", (long long)i);
    Scales sc;
    MNX_REQUIRE(bounds(a, sc), "muon: the iteration diverges with coefficients (%g, %g, %g)", a.coefficients[0],
                a.coefficients[1], a.coefficients[2]);
    Plan plan[2];
    for (int k = 0; k < 2; ++k) {
        if (int rc = lay_out(a, kForms[k].small, static_cast<char*>(a.workspace), plan[k])) return rc;
        if (!plan[k].mat.empty() && (!a.workspace || a.workspace_bytes < plan[k].bytes))
            return set_error(MNX_ERR_WORKSPACE, "muon: workspace too small");
    }
    for (int k = 0; k < 2; ++k)
        if (int rc = kForms[k].run(a, plan[k], sc, stream)) return rc;
    return MNX_OK;
}

}  // extern "C"
