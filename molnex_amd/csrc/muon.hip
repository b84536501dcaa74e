// Orthogonalised updates: the Newton-Schulz iteration of many matrices at once, and the Muon step around it.
//
//   m = m + (1 - mu) (g - m),  u = g + mu (m - g) with Nesterov's form, m without     (g negated to maximise)
//   X = u / max(|u|, eps), the Frobenius norm; transposed where it has more rows than columns: X is r x c, r <= c
//   steps times:  A = X X^T,  B = b A + c A A,  X = a X + B X
//   p = (1 - lr wd) p - lr s X,  s by the matrix's shape
//
// Numbers: X, A and B lie in the workspace as float16 scaled by powers of two, and are multiplied on the matrix cores
// with float32 sums.  Their entries are bounded by the iteration itself (|X|_2 <= max p(s) over the singular values
// that can occur, about 1.2 with the usual coefficients), so one scale a step, chosen on the host from the
// coefficients, keeps them inside float16's range with 11 bits each, where bfloat16 would keep 8: every rounding in
// the chain is 8 times finer at the same rate, and together they stay below bfloat16's own.  The first X is u itself
// times a power of two, exact for bfloat16 inputs; what remains of 1 / |u| (a factor from 1 to 2) goes into the first
// step's sums.  For float32 and float16 matrices every number is a pair hi + lo of float16, 22 bits, and a product is
// the three sums lo hi + hi lo + hi hi, in this order (lo lo is below 2^-22): with single ones a float16 result of
// 333 x 1234 was off by 1.2e-3, six times its rounding.
//
// All matrices of a call share each launch; a table in the workspace, written by a first small kernel from its
// arguments, tells a workgroup its matrix and tile.  Rows and columns are padded with zeros to multiples of 128, so
// that no load or store of the products has a bound to check.  A and B are symmetric: only tiles on and below the
// diagonal are formed, each stored twice.
#include "elem.h"

#include <cmath>
#include <type_traits>
#include <vector>

namespace mnx {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kPad = 128;  // sides of the padded matrices are multiples of it
constexpr int kChunk = 4096;  // elements of a matrix that a workgroup of the momentum kernel takes
constexpr int kCast = 64;     // side of the cast kernel's tiles
constexpr int kTableArgs = 24;

// One tensor: `batch` matrices of rows x cols.
struct Mat {
    void* p;         // parameters, or where the orthogonalised matrices go
    const void* g;   // gradients, or the matrices to orthogonalise
    float* m;        // momenta, or null
    _Float16* x[2];  // [planes][batch][rp][cp]
    _Float16* a;     // [planes][batch][rp][rp]
    _Float16* b;
    int64_t xplane, aplane;  // elements of a plane
    int32_t rows, cols, r, c, rp, cp, batch, dtype;
    float adjust;    // s
    uint32_t stat0;  // the first matrix's place among the norms
    uint32_t chunk0, cast0, sym0, upd0;  // first workgroup of each kind
};
// what follows a tensor's own units: entry `count` of each prefix
struct Prefix {
    uint32_t chunk, cast, sym, upd;
};

struct TableArgs {
    Mat mat[kTableArgs];
    int count, first;
};
static_assert(sizeof(TableArgs) <= 3840, "4 KB of arguments");

__global__ void __launch_bounds__(256) k_muon_table(TableArgs t, Mat* __restrict__ table) {
    const int words = t.count * int(sizeof(Mat) / 4);
    const uint32_t* from = reinterpret_cast<const uint32_t*>(t.mat);
    uint32_t* to = reinterpret_cast<uint32_t*>(table + t.first);
    for (int i = threadIdx.x; i < words; i += 256) to[i] = from[i];
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

__device__ __forceinline__ float load_any(const void* p, int64_t i, int dtype) { return load_elem(p, i, dtype); }

// The gradient, and the momentum after this step.
__device__ __forceinline__ float direction(float g, float m, const Momentum& h) {
    return h.nesterov ? h.w * g + h.mu * m : m;
}

// Momenta, and a partial sum of squares for each chunk of a matrix (float64: squares of any float32).
__global__ void __launch_bounds__(256) k_muon_momentum(const Mat* __restrict__ table, int count, Momentum h,
                                                       double* __restrict__ partial) {
    const uint32_t unit = blockIdx.x;
    const int at = find_mat(table, count, &Mat::chunk0, unit);
    const Mat& t = table[at];
    const int64_t n = int64_t(t.rows) * t.cols;
    const uint32_t per = uint32_t((n + kChunk - 1) / kChunk), u = unit - t.chunk0;
    const uint32_t which = u / per;
    const int64_t lo = int64_t(u - which * per) * kChunk, hi = min(lo + kChunk, n), off = which * n;
    double sum = 0;
    for (int64_t i = lo + threadIdx.x; i < hi; i += 256) {
        float v = load_any(t.g, off + i, t.dtype);
        if (t.m) {
            if (h.maximize) v = -v;
            const float m = t.m[off + i] * h.mu + h.w * v;
            t.m[off + i] = m;
            v = direction(v, m, h);
        }
        sum += double(v) * double(v);
    }
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    __shared__ double part[4];
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) partial[unit] = (part[0] + part[1]) + (part[2] + part[3]);
}

// The norm of each matrix: a wavefront a matrix.
__global__ void __launch_bounds__(64) k_muon_norm(const Mat* __restrict__ table, int count,
                                                  const double* __restrict__ partial, double eps,
                                                  Stat* __restrict__ stats) {
    const int at = find_mat(table, count, &Mat::stat0, blockIdx.x);
    const Mat& t = table[at];
    const uint32_t per = uint32_t((int64_t(t.rows) * t.cols + kChunk - 1) / kChunk);
    const double* mine = partial + t.chunk0 + uint64_t(blockIdx.x - t.stat0) * per;
    double sum = 0;
    for (uint32_t i = threadIdx.x; i < per; i += 64) sum += mine[i];
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if (threadIdx.x) return;
    Stat s{0, 1.0f};
    const double norm = sqrt(sum);
    if (!(norm < HUGE_VAL)) s.rho = __builtin_nanf("");  // infinite or NaN somewhere: so is every result
    else if (norm > 0) {
        int e;
        frexp(norm, &e);  // norm = f 2^e, 1/2 <= f < 1
        s.exponent = 12 - e;
        s.rho = float(ldexp(1.0, 12 - s.exponent) / fmax(norm, eps));  // 1 to 2 for a norm of eps or more
    }
    stats[blockIdx.x] = s;
}

template <int PL>
__device__ __forceinline__ void put(_Float16* to, int64_t plane, float v) {
    const _Float16 hi = _Float16(v);
    to[0] = hi;
    if constexpr (PL == 2) to[plane] = _Float16(v - float(hi));
}

// u in the products' layout, zeros around it.
template <int PL>
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
    for (int k = threadIdx.x; k < kCast * kCast; k += 256) {
        const int i = i0 + k / kCast, j = j0 + k % kCast;
        float v = 0;
        if (i < t.rows && j < t.cols) {
            const int64_t e = off + int64_t(i) * t.cols + j;
            v = load_any(t.g, e, t.dtype);
            if (t.m) {
                if (h.maximize) v = -v;
                v = direction(v, t.m[e], h);
            }
            v = ldexpf(v, s.exponent);
        }
        tile[k / kCast][k % kCast] = v;
    }
    __syncthreads();
    _Float16* x = t.x[0] + int64_t(which) * t.rp * t.cp;
    for (int k = threadIdx.x; k < kCast * kCast; k += 256) {
        const int i = k / kCast, j = k % kCast;
        put<PL>(x + int64_t(r0 + i) * t.cp + c0 + j, t.xplane, tall ? tile[j][i] : tile[i][j]);
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

// 16 bytes a lane from base + offset (bytes) to LDS, lane by lane from `to` on (M0).  In assembly, because for the builtin
// the compiler waits for every such load before the next read of LDS, also of other memory there.  The caller waits
// (vmcnt) and has a barrier before anyone reads what has come, and before it ends.
__device__ __forceinline__ void load_lds(const _Float16* base, uint32_t offset, _Float16* to) {
    const uint32_t m0 = uint32_t(uintptr_t((__attribute__((address_space(3))) _Float16*)to));
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(m0), "v"(offset), "s"(base)
                 : "memory", "m0");
}

// Four columns (k, k + 4) of the transposed 16-bit read: see read_tr.
__device__ __forceinline__ half8 read_tr(const _Float16* lo, const _Float16* hi) {
    typedef __attribute__((address_space(3))) short4v* P;
    const short4v a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)lo), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)hi);
    const half4 x = __builtin_bit_cast(half4, a), y = __builtin_bit_cast(half4, b);
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Four values of the last X, at columns j of row i, go into the parameters (or are the result); `count` of them exist.
template <typename T, bool TALL>
__device__ __forceinline__ void apply(T* p, int cols, int i, int j, int count, float decay, float rate,
                                      const float (&v)[4]) {
    typedef T Four __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    const int64_t at = TALL ? int64_t(j) * cols + i : int64_t(i) * cols + j, step = TALL ? cols : 1;
    if (!TALL && count >= 4) {
        Four* q = reinterpret_cast<Four*>(p + at);
        Four o = {};
        if (decay != 0) o = *q;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = T(decay * float(o[e]) - rate * v[e]);
        *q = o;
        return;
    }
    float old[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) old[e] = decay != 0 && e < count ? float(p[at + e * step]) : 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < count) p[at + e * step] = T(decay * old[e] - rate * v[e]);
}

constexpr int kKC = 64;  // k of a chunk

// A BT x BT tile of one product, the sum over k of I[i][k] J[j][k] (rows of both in memory), or with TR of I[i][k] J[k][j].
// Four wavefronts share it, a quarter each.  Chunks go from memory straight to LDS, 16 bytes a lane, into two buffers.
// Within a row of LDS the 16-byte pieces are permuted (by the lanes' source addresses: LDS itself is filled in lane order)
// so that the reads, 16 bytes of 16 rows or 64 bytes of 4 rows, meet every bank once.
//
// Operands of the next 16 k are read from LDS between the products of these.  The one barrier of a chunk stands before its
// last 16 k: by then every read of this buffer has come back and the next chunk has arrived, so behind it half the loads
// of the chunk after next and the first reads of the next run between those products, the other half of the loads between
// the next chunk's first ones.
//
// The last tile of a row or column may reach past the padded matrix: it reads what lies behind it in the workspace (rows
// and columns of the result that are not stored) and stores none of that.
template <int MODE, int PL, int BT>
__global__ void __launch_bounds__(256, BT == 128 ? 2 : 1) k_muon_product(const Mat* __restrict__ table, int count,
                                                                        uint32_t units, Step s,
                                                                        const Stat* __restrict__ stats, Apply ap) {
    constexpr bool SYM = MODE == kGram || MODE == kPoly, TR = !SYM;
    constexpr int W = BT / 2, MT = W / 32;  // a wavefront's part
    constexpr int SEG = PL == 1 ? 1 : 3;
    constexpr int FETCH = BT / 32;  // loads a lane of either operand's chunk
    constexpr int PIECES = BT / 8;  // of a sum's columns
    __shared__ _Float16 sI0[BT * kKC], sI1[BT * kKC], sJ0[BT * kKC], sJ1[BT * kKC];
    const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = wave & 1, wj = wave >> 1;
    const uint32_t per = (units + 7) / 8;
    uint32_t u = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
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
    const int K = MODE == kGram ? t.cp : t.rp;
    const _Float16* X = t.x[s.from] + int64_t(which) * t.rp * t.cp;
    const _Float16* A = t.a + int64_t(which) * t.rp * t.rp;
    const _Float16* B = t.b + int64_t(which) * t.rp * t.rp;
    const _Float16* I = (MODE == kGram ? X : MODE == kPoly ? A : B) + int64_t(ti) * BT * K;
    const int64_t iplane = MODE == kGram ? t.xplane : t.aplane;
    const _Float16* J = TR ? X + tj * BT : (MODE == kGram ? X : A) + int64_t(tj) * BT * K;
    const int64_t jplane = MODE == kPoly ? t.aplane : t.xplane;

    f32x16 acc[MT][MT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < MT; ++n)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[m][n][q] = 0.f;

    const int per_seg = K / kKC, chunks = SEG * per_seg;
    // a wavefront fills 1 KB of LDS at a time, every fourth: 8 rows of 64 k, or sums' columns piece after piece
    const int frow = wave * 8 + (lane >> 3);
    const uint32_t irow = 2 * (uint32_t(frow) * K + (((lane & 7) ^ ((frow >> 1) & 7)) << 3));  // bytes
    const int64_t istep = int64_t(32) * K;
    uint32_t jrow[TR ? FETCH : 1];
    if constexpr (TR) {
#pragma unroll
        for (int n = 0; n < FETCH; ++n) {
            const int piece = (n * 4 + wave) * 64 + lane, k = piece / PIECES, c = piece % PIECES;
            const int turn = BT == 192 ? ((k >> 1) & 1) << 2 : (k & 3) << 2;
            jrow[n] = 2 * (uint32_t(k) * t.cp + ((c ^ turn) << 3));
        }
    }
    struct Source {
        const _Float16 *i, *j;
    };
    auto source = [&](int chunk) {
        Source f{I, J};
        if constexpr (PL == 2) {
            const int seg = chunk >= 2 * per_seg ? 2 : chunk >= per_seg ? 1 : 0;
            chunk -= seg * per_seg;
            if (seg == 0) f.i += iplane;
            if (seg == 1) f.j += jplane;
        }
        f.i += chunk * kKC;
        f.j += TR ? int64_t(chunk * kKC) * t.cp : chunk * kKC;
        return f;
    };
    // the n-th of a chunk's 2 FETCH loads
    auto fetch = [&](const Source& f, int n, _Float16* bi, _Float16* bj) {
        if (n < FETCH) load_lds(f.i + n * istep, irow, bi + (n * 4 + wave) * 512);
        else if constexpr (TR) load_lds(f.j, jrow[n - FETCH], bj + ((n - FETCH) * 4 + wave) * 512);
        else load_lds(f.j + (n - FETCH) * istep, irow, bj + ((n - FETCH) * 4 + wave) * 512);
    };
    struct Frags {
        half8 i[MT], j[MT];
    };
    const int ki = (wi * W + l32) * kKC, kj = (wj * W + l32) * kKC, turn = (l32 >> 1) & 7;  // 32 rows on turn alike
    const int trow = 8 * half + ((lane & 15) >> 2), tcol = wj * W + (l32 & 16) + (lane & 3) * 4;
    const int tturn = BT == 192 ? ((trow >> 1) & 1) << 2 : (trow & 3) << 2;
    auto read_i = [&](int m, int ks, const _Float16* bi) {
        return *reinterpret_cast<const half8*>(bi + ki + m * 32 * kKC + (((2 * ks + half) ^ turn) << 3));
    };
    auto read_j = [&](int n, int ks, const _Float16* bj) {
        if constexpr (!TR) {
            return *reinterpret_cast<const half8*>(bj + kj + n * 32 * kKC + (((2 * ks + half) ^ turn) << 3));
        } else {
            const int col = tcol + n * 32;
            const _Float16* q = bj + (16 * ks + trow) * BT + (((col >> 3) ^ tturn) << 3) + (col & 4);
            return read_tr(q, q + 4 * BT);  // four sums on turn alike
        }
    };
    // The products of `now`, with the reads of `next` and `loads` between them.
    auto multiply = [&](const Frags& now, Frags& next, int ks, const _Float16* bi, const _Float16* bj, auto loads) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            next.j[m] = read_j(m, ks, bj);
            next.i[m] = read_i(m, ks, bi);
            loads(m);
#pragma unroll
            for (int n = 0; n < MT; ++n) acc[m][n] = mfma(now.j[n], now.i[m], acc[m][n]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto arrived = [] {  // everyone's loads and reads
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    Frags f0, f1;
    // Chunk c in (bi, bj), its first operands in f0; (oi, oj) takes or holds the next.  REST: the second half of the next
    // chunk's loads is still to come; MORE: a chunk after next begins.
    auto body = [&](int c, _Float16* bi, _Float16* bj, _Float16* oi, _Float16* oj, auto rest, auto more) {
        const auto nothing = [](int) {};
        if constexpr (rest) {
            const Source f = source(c + 1);
            multiply(f0, f1, 1, bi, bj, [&](int m) {
#pragma unroll
                for (int n = 0; n < FETCH / MT; ++n) fetch(f, FETCH + m * (FETCH / MT) + n, oi, oj);
            });
        } else {
            multiply(f0, f1, 1, bi, bj, nothing);
        }
        multiply(f1, f0, 2, bi, bj, nothing);
        multiply(f0, f1, 3, bi, bj, nothing);
        arrived();
        if constexpr (more) {
            const Source f = source(c + 2);
            multiply(f1, f0, 0, oi, oj, [&](int m) {
#pragma unroll
                for (int n = 0; n < FETCH / MT; ++n) fetch(f, m * (FETCH / MT) + n, bi, bj);
            });
        } else {
            multiply(f1, f0, 0, oi, oj, nothing);  // after the last chunk, reads of the one before that nobody uses
        }
    };
    const std::true_type yes;
    const std::false_type no;
    {
        const Source f = source(0), g = source(1);
#pragma unroll
        for (int n = 0; n < 2 * FETCH; ++n) fetch(f, n, sI0, sJ0);
        arrived();
#pragma unroll
        for (int n = 0; n < FETCH; ++n) fetch(g, n, sI1, sJ1);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            f0.i[m] = read_i(m, 0, sI0);
            f0.j[m] = read_j(m, 0, sJ0);
        }
    }
    int c = 0;  // chunks are an even number: K is a multiple of 128
    for (; c + 2 < chunks; c += 2) {
        body(c, sI0, sJ0, sI1, sJ1, yes, yes);
        body(c + 1, sI1, sJ1, sI0, sJ0, yes, yes);
    }
    body(c, sI0, sJ0, sI1, sJ1, yes, no);
    body(c + 1, sI1, sJ1, sI0, sJ0, no, no);

    // acc[m][n][q] belongs to row i = 32 m + l32 and column j = 32 n + 8 (q / 4) + 4 half + q % 4 of the wave's part
    float own = s.own, prod = s.prod;
    if (s.first) {
        const float rho = stats[t.stat0 + which].rho;
        if (MODE == kGram) prod *= rho * rho;
        if (MODE == kUpdate || MODE == kFinal) {
            own *= rho;
            prod *= rho;
        }
    }
    const int64_t ld = SYM ? t.rp : t.cp;
    const int64_t oplane = SYM ? t.aplane : t.xplane;
    const _Float16* E = MODE == kPoly ? A : X;
    _Float16* out = (MODE == kGram ? t.a : MODE == kPoly ? t.b : t.x[s.from ^ 1]) + int64_t(which) * t.rp * ld;
    const int i0 = ti * BT + wi * W + l32, j0 = tj * BT + wj * W + 4 * half;
    const int rows = MODE == kFinal ? t.r : t.rp, cols = MODE == kFinal ? t.c : SYM ? t.rp : t.cp;
    float decay = 0, rate = -ap.inv;  // of p and of its change; the result itself has no p
    if (MODE == kFinal && t.m) {
        const float lr = ap.lr_device ? *ap.lr_device : ap.lr;
        decay = 1 - lr * ap.wd;
        rate = lr * t.adjust * ap.inv;
    }
    // every four consecutive columns of a row
    auto each = [&](auto store) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < MT; ++n)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int i = i0 + m * 32, j = j0 + n * 32 + 8 * q;
                    if (i >= rows || j >= cols) continue;
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = prod * acc[m][n][4 * q + e];
                    if constexpr (MODE != kGram) {
#pragma unroll
                        for (int pl = PL - 1; pl >= 0; --pl) {
                            const half4 old = *reinterpret_cast<const half4*>(E + pl * oplane + int64_t(i) * ld + j);
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[e] += own * float(old[e]);
                        }
                    }
                    store(i, j, v);
                }
    };
    if constexpr (MODE == kFinal) {
        auto as = [&](auto type, auto tall) {
            auto* p = static_cast<decltype(type)*>(t.p) + int64_t(which) * t.rows * t.cols;
            each([&](int i, int j, const float (&v)[4]) {
                apply<decltype(type), decltype(tall)::value>(p, t.cols, i, j, cols - j, decay, rate, v);
            });
        };
        const bool tall = t.rows > t.cols;
        if constexpr (PL == 1) {
            if (tall) as(__bf16{}, yes);
            else as(__bf16{}, no);
        } else if (t.dtype == kF32) {
            if (tall) as(float{}, yes);
            else as(float{}, no);
        } else {
            if (tall) as(_Float16{}, yes);
            else as(_Float16{}, no);
        }
    } else {
        each([&](int i, int j, const float (&v)[4]) {
            half4 hi, lo;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                hi[e] = _Float16(v[e]);
                lo[e] = _Float16(v[e] - float(hi[e]));
            }
            *reinterpret_cast<half4*>(out + int64_t(i) * ld + j) = hi;
            if constexpr (PL == 2) *reinterpret_cast<half4*>(out + oplane + int64_t(i) * ld + j) = lo;
            if (SYM && ti != tj) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int64_t mirror = int64_t(j + e) * ld + i;
                    out[mirror] = hi[e];
                    if constexpr (PL == 2) out[oplane + mirror] = lo[e];
                }
            }
        });
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

constexpr int kTile[] = {256, 192, 128}, kTiles = 3;

// The time of a launch, about: rounds of the tiles that the card holds at once (256 CUs; two tiles of 128 a CU), by what a
// tile takes.
double cost(const std::vector<Mat>& mats, bool sym, int tile) {
    double tiles = 0;
    for (const Mat& t : mats) tiles += double(tiles_of(t, sym, tile));
    const double slots = tile == 128 ? 512 : 256, each = tile == 256 ? 4.0 : tile == 192 ? 2.4 : 2.2;
    return std::ceil(tiles / slots) * each;
}

// float16 numbers that stand for one of X, A and B
inline int planes_of(int dtype) { return dtype == kBF16 ? 1 : 2; }

// Lays the tensors of `planes` planes out over the workspace (from `base`, which may be null for its size alone).
int lay_out(const mnx_muon_args& a, int planes, char* base, Plan& plan) {
    Workspace ws{base, 0};
    uint64_t chunk = 0, cast = 0, stat = 0;
    for (int64_t i = 0; i < a.count; ++i) {
        if (planes_of(a.dtype[i]) != planes || !a.batch[i] || !a.rows[i] || !a.cols[i]) continue;
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
        t.xplane = a.batch[i] * t.rp * t.cp;
        t.aplane = a.batch[i] * t.rp * t.rp;
        t.stat0 = uint32_t(stat);
        t.chunk0 = uint32_t(chunk);
        t.cast0 = uint32_t(cast);
        const uint64_t b = uint64_t(a.batch[i]);
        stat += b;
        chunk += b * uint64_t(ceil_div(int64_t(t.rows) * t.cols, kChunk));
        cast += b * uint64_t(t.rp / kCast) * (t.cp / kCast);
        for (_Float16*& x : t.x) x = ws.take<_Float16>(size_t(planes * t.xplane));
        t.a = ws.take<_Float16>(size_t(planes * t.aplane));
        t.b = ws.take<_Float16>(size_t(planes * t.aplane));
        // a grid has fewer than 2^32 threads
        MNX_REQUIRE(std::max({chunk, cast, stat}) < (1u << 23), "muon: too many matrices in one call");
        plan.mat.push_back(t);
    }
    for (int kind = 0; kind < 2; ++kind) {
        int best = 0;
        for (int k = 1; k < kTiles; ++k)
            if (cost(plan.mat, kind == 0, kTile[k]) < cost(plan.mat, kind == 0, kTile[best])) best = k;
        (kind == 0 ? plan.sym_tile : plan.upd_tile) = kTile[best];
    }
    uint64_t sym = 0, upd = 0;
    for (Mat& t : plan.mat) {
        t.sym0 = uint32_t(sym);
        t.upd0 = uint32_t(upd);
        sym += tiles_of(t, true, plan.sym_tile);
        upd += tiles_of(t, false, plan.upd_tile);
    }
    plan.total = {uint32_t(chunk), uint32_t(cast), uint32_t(sym), uint32_t(upd)};
    // the last tiles read past the last matrix
    int64_t past = 0;
    for (const Mat& t : plan.mat) past = std::max<int64_t>(past, int64_t(256) * t.cp);
    if (past) ws.take<_Float16>(size_t(past));
    plan.stats = uint32_t(stat);
    plan.partial = ws.take<double>(size_t(chunk));
    plan.stat = ws.take<Stat>(size_t(stat));
    plan.table = ws.take<Mat>(plan.mat.size());
    plan.bytes = ws.used;
    return MNX_OK;
}

template <int MODE, int PL>
int product(const Plan& plan, const Step& s, const Apply& ap, mnx_stream_t stream) {
    constexpr bool SYM = MODE == kGram || MODE == kPoly;
    const int tile = SYM ? plan.sym_tile : plan.upd_tile;
    const uint32_t units = SYM ? plan.total.sym : plan.total.upd, grid = uint32_t(up(units, 8));
    const int count = int(plan.mat.size());
    const auto kernel = tile == 256 ? k_muon_product<MODE, PL, 256>
                                    : tile == 192 ? k_muon_product<MODE, PL, 192> : k_muon_product<MODE, PL, 128>;
    kernel<<<grid, 256, 0, stream>>>(plan.table, count, units, s, plan.stat, ap);
    MNX_CHECK_LAUNCH();
    return MNX_OK;
}

template <int PL>
int run(const mnx_muon_args& a, const Plan& plan, const Scales& sc, mnx_stream_t stream) {
    const int count = int(plan.mat.size());
    if (!count) return MNX_OK;
    for (int at = 0; at < count; at += kTableArgs) {
        TableArgs t;
        t.first = at;
        t.count = std::min(kTableArgs, count - at);
        for (int i = 0; i < t.count; ++i) t.mat[i] = plan.mat[size_t(at + i)];
        k_muon_table<<<1, 256, 0, stream>>>(t, plan.table);
        MNX_CHECK_LAUNCH();
    }
    const Momentum h{float(a.momentum), float(1 - a.momentum), a.nesterov, a.maximize};
    k_muon_momentum<<<plan.total.chunk, 256, 0, stream>>>(plan.table, count, h, plan.partial);
    MNX_CHECK_LAUNCH();
    k_muon_norm<<<plan.stats, 64, 0, stream>>>(plan.table, count, plan.partial, a.eps, plan.stat);
    MNX_CHECK_LAUNCH();
    k_muon_cast<PL><<<plan.total.cast, 256, 0, stream>>>(plan.table, count, h, plan.stat);
    MNX_CHECK_LAUNCH();
    const double ca = a.coefficients[0], cb = a.coefficients[1], cc = a.coefficients[2];
    const Apply none{};
    for (int k = 0; k < a.steps; ++k) {
        const double A = sc.a[k], B = sc.b[k];
        const int from = k & 1, first = k == 0, last = k + 1 == a.steps;
        const double xs = first ? 4096.0 : sc.x[k];  // the first X is stored at 2^12 whatever the bounds say
        const Step gram{0.f, float(A / (xs * xs)), from, first};
        const Step poly{float(B * cb / A), float(B * cc / (A * A)), from, first};
        const double to = last ? 1.0 : sc.x[k + 1];
        const Step update{float(to * ca / xs), float(to / (B * xs)), from, first};
        if (int rc = product<kGram, PL>(plan, gram, none, stream)) return rc;
        if (int rc = product<kPoly, PL>(plan, poly, none, stream)) return rc;
        const Apply ap{float(a.lr), a.lr_device, float(a.weight_decay), 1.0f};
        if (int rc = last ? product<kFinal, PL>(plan, update, ap, stream) : product<kUpdate, PL>(plan, update, none, stream))
            return rc;
    }
    return MNX_OK;
}

}  // namespace
}  // namespace mnx

using namespace mnx;

extern "C" {

size_t mnx_muon_workspace_bytes(const mnx_muon_args* args) {
    clear_error();
    if (!args || check_args(*args) != MNX_OK) return 0;
    size_t most = 256;
    for (int planes = 1; planes <= 2; ++planes) {
        Plan plan;
        if (lay_out(*args, planes, nullptr, plan) != MNX_OK) return 0;
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
    for (int planes = 1; planes <= 2; ++planes) {
        if (int rc = lay_out(a, planes, static_cast<char*>(a.workspace), plan[planes - 1])) return rc;
        if (!plan[planes - 1].mat.empty() && (!a.workspace || a.workspace_bytes < plan[planes - 1].bytes))
            return set_error(MNX_ERR_WORKSPACE, "muon: workspace too small");
    }
    if (int rc = run<1>(a, plan[0], sc, stream)) return rc;
    return run<2>(a, plan[1], sc, stream);
}

}  // extern "C"
