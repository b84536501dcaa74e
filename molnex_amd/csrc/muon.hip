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
#include <vector>

namespace mnx {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kPad = 128;
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

__device__ __forceinline__ void load_lds(const _Float16* from, _Float16* to) {
    __builtin_amdgcn_global_load_lds(
        const_cast<__attribute__((address_space(1))) void*>((const __attribute__((address_space(1))) void*)from),
        (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// Four columns (k, k + 4) of the transposed 16-bit read: see read_tr.
__device__ __forceinline__ half8 read_tr(const _Float16* lo, const _Float16* hi) {
    typedef __attribute__((address_space(3))) short4v* P;
    const short4v a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)lo), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)hi);
    const half4 x = __builtin_bit_cast(half4, a), y = __builtin_bit_cast(half4, b);
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
}

constexpr int kKC = 64;  // k of a chunk

// A tile of I rows against J columns of one product, sum over k of I[i][k] J[j][k] (rows of both in memory), or with TR
// of I[i][k] J[k][j].  Tiles go from memory straight to LDS, 16 bytes a lane, one chunk ahead.  Within a row of LDS the
// 16-byte pieces are permuted (by the lanes' source addresses: LDS itself is filled in lane order) so that the reads,
// 16 bytes of 32 rows or 64 bytes of 4 rows, meet every bank once.
template <int MODE, int PL, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__((BM / WM) * (BN / WN) * 64) k_muon_product(const Mat* __restrict__ table, int count,
                                                                           uint32_t units, Step s,
                                                                           const Stat* __restrict__ stats, Apply ap) {
    constexpr bool SYM = MODE == kGram || MODE == kPoly, TR = !SYM;
    constexpr int WAVES = (BM / WM) * (BN / WN), MT = WM / 32, NT = WN / 32;
    constexpr int SEG = PL == 1 ? 1 : 3;
    __shared__ _Float16 sI[2][BM * kKC], sJ[2][BN * kKC];
    const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = wave % (BM / WM), wj = wave / (BM / WM);
    const uint32_t per = (units + 7) / 8;
    uint32_t u = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (u >= units) return;
    const int at = find_mat(table, count, SYM ? &Mat::sym0 : &Mat::upd0, u);
    const Mat& t = table[at];
    u -= SYM ? t.sym0 : t.upd0;
    const int ni = t.rp / BM, nj = t.cp / BN;
    const uint32_t tiles = SYM ? uint32_t(ni * (ni + 1) / 2) : uint32_t(ni * nj);
    const uint32_t which = u / tiles;
    u -= which * tiles;
    int ti, tj;
    if (SYM) {
        ti = int((sqrtf(8.0f * float(u) + 1.0f) - 1.0f) * 0.5f);
        while (uint32_t(ti * (ti + 1) / 2) > u) --ti;
        while (uint32_t((ti + 1) * (ti + 2) / 2) <= u) ++ti;
        tj = int(u) - ti * (ti + 1) / 2;
    } else {
        tj = int(u) / ni;
        ti = int(u) - tj * ni;
    }
    ti = __builtin_amdgcn_readfirstlane(ti);
    tj = __builtin_amdgcn_readfirstlane(tj);
    const int K = MODE == kGram ? t.cp : t.rp;
    const _Float16* X = t.x[s.from] + int64_t(which) * t.rp * t.cp;
    const _Float16* A = t.a + int64_t(which) * t.rp * t.rp;
    const _Float16* B = t.b + int64_t(which) * t.rp * t.rp;
    const _Float16* I = (MODE == kGram ? X : MODE == kPoly ? A : B) + int64_t(ti) * BM * K;
    const int64_t iplane = MODE == kGram ? t.xplane : t.aplane;
    const _Float16* J = TR ? X + tj * BN : (MODE == kGram ? X : A) + int64_t(tj) * BN * K;
    const int64_t jplane = MODE == kPoly ? t.aplane : t.xplane;

    f32x16 acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[m][n][q] = 0.f;

    const int per_seg = K / kKC, chunks = SEG * per_seg;
    auto fetch = [&](int chunk, int buf) {
        int k0 = chunk;
        const _Float16 *i = I, *j = J;
        if constexpr (PL == 2) {
            const int seg = chunk >= 2 * per_seg ? 2 : chunk >= per_seg ? 1 : 0;
            k0 -= seg * per_seg;
            if (seg == 0) i += iplane;
            if (seg == 1) j += jplane;
        }
        k0 *= kKC;
#pragma unroll
        for (int n = wave; n < BM / 8; n += WAVES) {
            const int row = n * 8 + (lane >> 3);
            load_lds(i + int64_t(row) * K + k0 + (((lane & 7) ^ ((row >> 1) & 7)) << 3), &sI[buf][n * 512]);
        }
        if constexpr (!TR) {
#pragma unroll
            for (int n = wave; n < BN / 8; n += WAVES) {
                const int row = n * 8 + (lane >> 3);
                load_lds(j + int64_t(row) * K + k0 + (((lane & 7) ^ ((row >> 1) & 7)) << 3), &sJ[buf][n * 512]);
            }
        } else {
            constexpr int LPR = BN / 8;  // lanes of a row
#pragma unroll
            for (int n = wave; n < BN / 8; n += WAVES) {
                const int k = n * (64 / LPR) + lane / LPR;
                load_lds(j + int64_t(k0 + k) * t.cp + (((lane % LPR) ^ ((k & 3) << 2)) << 3), &sJ[buf][n * 512]);
            }
        }
    };
    fetch(0, 0);
    for (int chunk = 0; chunk < chunks; ++chunk) {
        __syncthreads();  // this chunk has arrived, and the other buffer is read
        if (chunk + 1 < chunks) fetch(chunk + 1, (chunk + 1) & 1);
        const _Float16 *pi = sI[chunk & 1], *pj = sJ[chunk & 1];
#pragma unroll
        for (int ks = 0; ks < kKC / 16; ++ks) {
            half8 fi[MT], fj[NT];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const int row = wi * WM + m * 32 + l32;
                fi[m] = *reinterpret_cast<const half8*>(pi + row * kKC + (((2 * ks + half) ^ ((row >> 1) & 7)) << 3));
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if constexpr (!TR) {
                    const int row = wj * WN + n * 32 + l32;
                    fj[n] = *reinterpret_cast<const half8*>(pj + row * kKC + (((2 * ks + half) ^ ((row >> 1) & 7)) << 3));
                } else {
                    const int k = 16 * ks + 8 * half + ((lane & 15) >> 2);
                    const int col = wj * WN + n * 32 + (l32 & 16) + (lane & 3) * 4;
                    const _Float16* q = pj + k * BN + (((col >> 3) ^ ((k & 3) << 2)) << 3) + (col & 4);
                    fj[n] = read_tr(q, q + 4 * BN);
                }
            }
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n) acc[m][n] = mfma(fj[n], fi[m], acc[m][n]);
        }
    }

    // acc[m][n][q] belongs to row i = 32 m + l32 and column j = 32 n + 8 (q / 4) + 4 half + q % 4 of the wave's tile
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
    float decay = 1, rate = -ap.inv;  // rate: of p's change, or of the result itself
    if (MODE == kFinal && t.m) {
        const float lr = ap.lr_device ? *ap.lr_device : ap.lr;
        decay = 1 - lr * ap.wd;
        rate = lr * t.adjust * ap.inv;
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int i = ti * BM + wi * WM + m * 32 + l32;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int j = tj * BN + wj * WN + n * 32 + 8 * q + 4 * half;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = prod * acc[m][n][4 * q + e];
                const int64_t place = int64_t(i) * ld + j;
                if constexpr (MODE != kGram) {
#pragma unroll
                    for (int pl = PL - 1; pl >= 0; --pl) {
                        const half4 old = *reinterpret_cast<const half4*>(E + pl * oplane + place);
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] += own * float(old[e]);
                    }
                }
                if constexpr (MODE == kFinal) {
                    if (i >= t.r) continue;
                    const bool tall = t.rows > t.cols;
                    const int64_t off = int64_t(which) * t.rows * t.cols;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (j + e >= t.c) continue;
                        const int64_t at = off + (tall ? int64_t(j + e) * t.cols + i : int64_t(i) * t.cols + j + e);
                        const float old = t.m ? decay * load_any(t.p, at, t.dtype) : 0.f;
                        store_elem(t.p, at, t.dtype, old - rate * v[e]);
                    }
                } else {
                    half4 hi, lo;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        hi[e] = _Float16(v[e]);
                        lo[e] = _Float16(v[e] - float(hi[e]));
                    }
                    *reinterpret_cast<half4*>(out + place) = hi;
                    if constexpr (PL == 2) *reinterpret_cast<half4*>(out + oplane + place) = lo;
                    if (SYM && ti != tj) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int64_t mirror = int64_t(j + e) * ld + i;
                            out[mirror] = hi[e];
                            if constexpr (PL == 2) out[oplane + mirror] = lo[e];
                        }
                    }
                }
            }
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

// float16 numbers that stand for one of X, A and B
inline int planes_of(int dtype) { return dtype == kBF16 ? 1 : 2; }

// Lays the tensors of `planes` planes out over the workspace (from `base`, which may be null for its size alone).
int lay_out(const mnx_muon_args& a, int planes, char* base, Plan& plan) {
    Workspace ws{base, 0};
    uint64_t chunk = 0, cast = 0, sym = 0, upd = 0, stat = 0;
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
        t.sym0 = uint32_t(sym);
        t.upd0 = uint32_t(upd);
        const uint64_t b = uint64_t(a.batch[i]), ni = t.rp / kPad, nj = t.cp / kPad;
        stat += b;
        chunk += b * uint64_t(ceil_div(int64_t(t.rows) * t.cols, kChunk));
        cast += b * uint64_t(t.rp / kCast) * (t.cp / kCast);
        sym += b * (ni * (ni + 1) / 2);
        upd += b * ni * nj;
        for (_Float16*& x : t.x) x = ws.take<_Float16>(size_t(planes * t.xplane));
        t.a = ws.take<_Float16>(size_t(planes * t.aplane));
        t.b = ws.take<_Float16>(size_t(planes * t.aplane));
        // a grid has fewer than 2^32 threads
        MNX_REQUIRE(std::max({chunk, cast, sym, upd, stat}) < (1u << 23), "muon: too many matrices in one call");
        plan.mat.push_back(t);
    }
    plan.total = {uint32_t(chunk), uint32_t(cast), uint32_t(sym), uint32_t(upd)};
    plan.stats = uint32_t(stat);
    plan.partial = ws.take<double>(size_t(chunk));
    plan.stat = ws.take<Stat>(size_t(stat));
    plan.table = ws.take<Mat>(plan.mat.size());
    plan.bytes = ws.used;
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
    const uint32_t gs = uint32_t(up(plan.total.sym, 8)), gu = uint32_t(up(plan.total.upd, 8));
    const Apply none{};
    for (int k = 0; k < a.steps; ++k) {
        const double x = sc.x[k], A = sc.a[k], B = sc.b[k];
        const int from = k & 1, first = k == 0;
        // the first X is stored at 2^12 whatever the bounds say
        const double xs = first ? 4096.0 : x;
        k_muon_product<kGram, PL, 128, 128, 64, 64><<<gs, 256, 0, stream>>>(
            plan.table, count, plan.total.sym, Step{0.f, float(A / (xs * xs)), from, first}, plan.stat, none);
        MNX_CHECK_LAUNCH();
        k_muon_product<kPoly, PL, 128, 128, 64, 64><<<gs, 256, 0, stream>>>(
            plan.table, count, plan.total.sym, Step{float(B * cb / A), float(B * cc / (A * A)), from, first}, plan.stat,
            none);
        MNX_CHECK_LAUNCH();
        const double to = k + 1 == a.steps ? 1.0 : sc.x[k + 1];
        const Step s{float(to * ca / xs), float(to / (B * xs)), from, first};
        if (k + 1 < a.steps) {
            k_muon_product<kUpdate, PL, 128, 128, 64, 64><<<gu, 256, 0, stream>>>(plan.table, count, plan.total.upd, s,
                                                                                plan.stat, none);
        } else {
            const Apply ap{float(a.lr), a.lr_device, float(a.weight_decay), 1.0f};
            k_muon_product<kFinal, PL, 128, 128, 64, 64><<<gu, 256, 0, stream>>>(plan.table, count, plan.total.upd, s,
                                                                               plan.stat, ap);
        }
        MNX_CHECK_LAUNCH();
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
