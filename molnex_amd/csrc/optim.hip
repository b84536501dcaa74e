// AdamW over many tensors, with 32-bit or 8-bit states, and the 2-norm of many tensors.
//
//   g' = s g, s = min(1, max_norm / (norm + 1e-6)) (1 without a max_norm);  t += 1
//   m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g' g'
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// The tensors' addresses travel in the kernels' arguments (a table of up to kTensors entries a launch), so a call
// copies nothing to the device and can be captured in a graph; the step counts t, the norm and what follows from
// them stay on the device.  A workgroup takes a chunk of one tensor, four elements a thread and vector.
//
// Bytes bound it: an element takes 28 (32-bit states, float32) or 16 (8-bit) and 4 more for the norm.
//
// 8-bit states: 256 elements of a tensor share two bases (int16).  A code c stands for the float32 with the bits
// (base + c) << 20, exponent and 3 bits of mantissa, zero for c = 0: 7 bits of magnitude and a sign for m, 8 bits for
// v.  The base puts the block's largest magnitude, rounded up, at the largest code, so m reaches 2^-16 and v 2^-32 of
// it (sqrt(v) 2^-16).  Rounding is dithered: with b2 = 0.999 a step changes v by about 0.1 % where neighbouring codes
// are 6 to 12 % apart, and rounded to nearest the state would stand still.  The dither is a hash of (seed, tensor,
// step, element), so a run can be repeated bit for bit.  A v below the smallest code is rounded up to it: a zero
// there would leave m / eps.  Elements whose m or v is not finite are kept out of the base and read back as NaN.
//
// This file is compiled without contraction to fused multiply-adds: the states' bits decide their codes, and are
// those of the plain operations in float32.
#include "elem.h"

namespace mnx {

constexpr int kTensors = 64;       // tensors of one update launch: the table stays below 4 KB of arguments
constexpr int kNormTensors = 160;  // tensors of one norm launch
constexpr int kStepTensors = 480;  // tensors of one launch of the step counts, a thread each
constexpr int kBlock = 256;        // elements of a block of 8-bit states

// Elements that a workgroup takes.  The update reads all that its chunk has, two vectors of each array a thread, and is
// done: 128 M fp32 parameters take 645 us so, 656 us with four vectors, and 721 us in chunks of 8192 looped over; 24 M
// bf16 ones 95, 99 and 117 us, 64 M with 8-bit states 261, 269 and 282 us.
// The norm's workgroups leave a partial sum each, for one workgroup to add up, and take more; small calls are cut
// finer, so that they reach every compute unit.
constexpr int kUpdateVectors = 2, kUpdateChunk = kUpdateVectors * 1024;
inline int norm_chunk(int64_t total) {
    int chunk = 1024;
    while (chunk < 16384 && total / chunk > 2048) chunk *= 2;
    return chunk;
}

// Workgroups of a launch at most (of 256 threads each; a grid has fewer than 2^32 threads).
constexpr int64_t kMostChunks = int64_t(1) << 23;
static_assert(MNX_OPTIM_MAX_ELEMENTS / kUpdateChunk <= kMostChunks, "a tensor fits a launch");

// Calls that move more than the 256 MB cache holds pass it by: 128 M fp32 parameters take 645 us so against 788 us,
// 64 M with 8-bit states and their read-back 261 against 307 us; 3.2 M, which fit, 31.9 against 29.9 us.
constexpr int64_t kCacheBytes = int64_t(256) << 20;

struct AdamwTable {
    void* p[kTensors];
    const void* g[kTensors];
    void* m[kTensors];
    void* v[kTensors];
    int16_t* bases[kTensors];
    int64_t n[kTensors];
    uint32_t start[kTensors + 1];  // first chunk of each tensor
    uint8_t dtype[kTensors];
    int count, first;              // tensors here, number of the first one in the call
};

struct NormTable {
    const void* g[kNormTensors];
    int64_t n[kNormTensors];
    uint32_t start[kNormTensors + 1];
    uint8_t dtype[kNormTensors];
    int count, chunk;
    int64_t out;  // place of the first chunk's partial sum
};

struct StepTable {
    float* step[kStepTensors];
    int count, first;
};

// The arguments of a launch, with a few pointers and numbers beside the table.
static_assert(sizeof(AdamwTable) <= 3840 && sizeof(NormTable) <= 3840 && sizeof(StepTable) <= 3856,
              "4 KB of arguments");

struct Hyper {
    float b1, w1, b2, w2, eps;  // w = 1 - b
};

// What the update needs of one tensor.
struct TensorScalars {
    float size, inv_root;  // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
    float decay;           // 1 - lr wd
    uint32_t key;          // of the dither
};
// ... and of all of them.
struct CallScalars {
    float scale;  // of the gradients; negative to maximise
    int skip;
};

__device__ __forceinline__ int find_tensor(const uint32_t* start, int count, uint32_t chunk) {
    int at = 0;
    for (int base = 0; base < count; base += 64) {
        const int i = base + (threadIdx.x & 63);
        at += __popcll(__ballot(i < count && start[i] <= chunk));
    }
    return __builtin_amdgcn_readfirstlane(at - 1);
}

// Four consecutive elements, at the alignment of one; past `end` they are 0 and not stored.  NT: past the caches, where
// that is 16 bytes a lane (narrower ones lose by it).
template <int DT>
struct Four {
    typedef typename Elem<DT>::T T;
    typedef T Packed __attribute__((ext_vector_type(4), aligned(sizeof(T))));
};
template <int DT, bool NT = false>
__device__ __forceinline__ void load4(const void* base, int64_t e, int64_t end, float (&v)[4]) {
    const auto* p = static_cast<const typename Elem<DT>::T*>(base);
    if (e + 4 <= end) {
        typename Four<DT>::Packed t;
        const auto* q = reinterpret_cast<const typename Four<DT>::Packed*>(p + e);
        if constexpr (NT && DT == kF32) t = __builtin_nontemporal_load(q);
        else t = *q;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = float(t[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = e + k < end ? float(p[e + k]) : 0.0f;
    }
}
template <int DT, bool NT = false>
__device__ __forceinline__ void store4(void* base, int64_t e, int64_t end, const float (&v)[4]) {
    using T = typename Elem<DT>::T;
    auto* p = static_cast<T*>(base);
    if (e + 4 <= end) {
        typename Four<DT>::Packed t;
#pragma unroll
        for (int k = 0; k < 4; ++k) t[k] = T(v[k]);
        auto* q = reinterpret_cast<typename Four<DT>::Packed*>(p + e);
        if constexpr (NT && DT == kF32) __builtin_nontemporal_store(t, q);
        else *q = t;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (e + k < end) p[e + k] = T(v[k]);
    }
}

typedef uint32_t PackedU32 __attribute__((aligned(1)));
typedef uint32_t Bases __attribute__((aligned(2)));  // m's base in the low half, v's in the high
__device__ __forceinline__ uint32_t load_codes(const uint8_t* p, int64_t e, int64_t end) {
    if (e + 4 <= end) return *reinterpret_cast<const PackedU32*>(p + e);
    uint32_t c = 0;
    for (int k = 0; k < 4; ++k)
        if (e + k < end) c |= uint32_t(p[e + k]) << 8 * k;
    return c;
}
__device__ __forceinline__ void store_codes(uint8_t* p, int64_t e, int64_t end, uint32_t c) {
    if (e + 4 <= end) {
        *reinterpret_cast<PackedU32*>(p + e) = c;
    } else {
        for (int k = 0; k < 4; ++k)
            if (e + k < end) p[e + k] = uint8_t(c >> 8 * k);
    }
}

// The chunk that a workgroup takes.
struct Chunk {
    int tensor;
    int64_t begin, end;
};
template <typename Table>
__device__ __forceinline__ Chunk chunk_at(const Table& t, uint32_t at, int chunk) {
    const int i = find_tensor(t.start, t.count, at);
    const int64_t begin = int64_t(at - t.start[i]) * chunk;
    return {i, begin, min(t.n[i], begin + chunk)};
}

// Sums over the workgroup, on every thread.
template <int THREADS>
__device__ __forceinline__ double block_sum(double v) {
    __shared__ double part[THREADS / 64];
    for (int off = 32; off; off >>= 1) v += __shfl_xor(v, off);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
    for (int i = 1; i < THREADS / 64; ++i) v += part[i];
    __syncthreads();
    return v;
}

// Squares are summed in float64: no overflow where the norm itself has none, and the same last bits whatever the
// order of the chunks.
template <int DT>
__device__ __forceinline__ double sum_squares(const void* g, const Chunk& c) {
    constexpr int U = 4;
    double s[U] = {};
    for (int64_t e = c.begin + threadIdx.x * 4; e < c.end; e += U * 1024) {
        float v[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u) load4<DT>(g, e + u * 1024, c.end, v[u]);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < 4; ++k) s[u] = __builtin_fma(double(v[u][k]), double(v[u][k]), s[u]);
    }
    return (s[0] + s[1]) + (s[2] + s[3]);
}

__global__ __launch_bounds__(256) void k_sumsq(const NormTable t, double* partial) {
    const Chunk c = chunk_at(t, blockIdx.x, t.chunk);
    const void* g = t.g[c.tensor];
    const int dt = t.dtype[c.tensor];
    const double s = block_sum<256>(dt == kF32    ? sum_squares<kF32>(g, c)
                                    : dt == kBF16 ? sum_squares<kBF16>(g, c)
                                                  : sum_squares<kF16>(g, c));
    if (threadIdx.x == 0) partial[t.out + blockIdx.x] = s;
}

__device__ __forceinline__ double sum_partial(const double* partial, int64_t chunks) {
    double s = 0;
#pragma unroll 8
    for (int64_t i = threadIdx.x; i < chunks; i += 1024) s += partial[i];
    return block_sum<1024>(s);
}

__global__ __launch_bounds__(1024) void k_norm(const double* partial, int64_t chunks, float* norm) {
    const double s = sum_partial(partial, chunks);
    if (threadIdx.x == 0) *norm = float(sqrt(s));
}

// A hash of 32-bit integers: multiplications by odd constants (the fractions of sqrt(2) and sqrt(3)) between shifted
// exclusive ors.
__device__ __forceinline__ uint32_t mix(uint32_t x) {
    x = (x ^ (x >> 15)) * 0x6A09E667u;
    x = (x ^ (x >> 13)) * 0xBB67AE85u;
    return x ^ (x >> 16);
}

// b^t of a whole number t by squaring, 24 multiplications deep at most.
__device__ __forceinline__ double power(double b, uint32_t t) {
    double r = 1;
    for (; t; t >>= 1, b *= b)
        if (t & 1) r *= b;
    return r;
}

// The step counts and everything that the update takes from them and from the norm, in float64.
__global__ __launch_bounds__(1024) void k_adamw_prepare(const StepTable t, const double* partial, int64_t chunks,
                                                       const float* norm_in, float* norm_out, double max_norm,
                                                       int skip_nonfinite, int maximize, double lr, const float* lr_dev,
                                                       double b1, double b2, double wd, uint32_t seed,
                                                       CallScalars* call, TensorScalars* tensors) {
    // what does not need the norm first, so that its loads and the sum's are on the way together
    const int i = threadIdx.x;
    float step = 0;
    TensorScalars s;
    if (i < t.count) {
        step = *t.step[i] + 1.0f;
        if (lr_dev) lr = *lr_dev;
        s.size = float(lr / (1 - power(b1, uint32_t(step))));
        s.inv_root = float(1 / sqrt(1 - power(b2, uint32_t(step))));
        s.decay = float(1 - lr * wd);
        s.key = mix(mix(seed * 0x3C6EF373u + uint32_t(t.first + i) * 0xA54FF53Bu) + uint32_t(step) * 0x510E527Fu);
    }
    double norm = 0;
    if (partial) norm = float(sqrt(sum_partial(partial, chunks)));
    else if (norm_in) norm = *norm_in;
    double scale = 1;
    if (max_norm >= 0) {
        scale = max_norm / (norm + 1e-6);
        if (scale >= 1) scale = 1;  // a NaN stays
    }
    const int skip = skip_nonfinite && !(fabs(norm) <= 3.402823466e38);
    if (threadIdx.x == 0) {
        call->scale = float(maximize ? -scale : scale);
        call->skip = skip;
        if (norm_out) *norm_out = float(norm);
    }
    if (skip || i >= t.count) return;
    *t.step[i] = step;
    tensors[t.first + i] = s;
}

struct Moments {
    float m, v;
};

__device__ __forceinline__ Moments moments(const Hyper& h, float m, float v, float g) {
    return {m * h.b1 + g * h.w1, v * h.b2 + (g * g) * h.w2};
}
// The formula's float32 operations, a unit of half a place each.  They are free beside 32-bit moments, whose bytes
// bound the kernel (k_adamw: 3.2 M elements 16.4 us with them and 16.3 with those below, 128 M 186 a launch with both).
__device__ __forceinline__ float updated(const Hyper& h, const TensorScalars& s, float p, const Moments& a) {
    return p * s.decay - s.size * a.m / (sqrtf(a.v) * s.inv_root + h.eps);
}
// Beside 8-bit moments, which know m to one part in 16 at best, the square root and the reciprocal are the hardware's
// instructions, a unit of the last place each: instructions bound that kernel (3.2 M elements 16.5 us with them and
// 18.0 with the exact forms, 64 M 94 against 103 a launch).
// The root's instruction takes no subnormals: a v below 2^-96 is scaled (its root is far below any eps but 0).
__device__ __forceinline__ float updated_fast(const Hyper& h, const TensorScalars& s, float p, const Moments& a) {
    const bool tiny = a.v < 0x1p-96f;
    const float root = __builtin_amdgcn_sqrtf(tiny ? a.v * 0x1p96f : a.v) * (tiny ? 0x1p-48f : 1.0f);
    return p * s.decay - s.size * a.m * __builtin_amdgcn_rcpf(root * s.inv_root + h.eps);
}

template <int DT, bool NT>
__device__ __forceinline__ void update32(const AdamwTable& t, const Chunk& c, const Hyper& h, const TensorScalars& s,
                                         float scale) {
    constexpr int U = kUpdateVectors;
    const void* gs = t.g[c.tensor];
    void *ps = t.p[c.tensor], *ms = t.m[c.tensor], *vs = t.v[c.tensor];
    const int64_t e = c.begin + threadIdx.x * 4;
    float p[U][4], g[U][4], m[U][4], v[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        load4<DT, NT>(gs, e + u * 1024, c.end, g[u]);
        load4<DT, NT>(ps, e + u * 1024, c.end, p[u]);
        load4<kF32, NT>(ms, e + u * 1024, c.end, m[u]);
        load4<kF32, NT>(vs, e + u * 1024, c.end, v[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const Moments a = moments(h, m[u][k], v[u][k], g[u][k] * scale);
            p[u][k] = updated(h, s, p[u][k], a);
            m[u][k] = a.m;
            v[u][k] = a.v;
        }
        store4<DT, NT>(ps, e + u * 1024, c.end, p[u]);
        store4<kF32, NT>(ms, e + u * 1024, c.end, m[u]);
        store4<kF32, NT>(vs, e + u * 1024, c.end, v[u]);
    }
}

// Chunks are taken from the last to the first: the norm read them from the first to the last, so the latest gradients
// are still in the 256 MB cache.
template <bool NT>
__global__ __launch_bounds__(256) void k_adamw(const AdamwTable t, const Hyper h, const CallScalars* call,
                                               const TensorScalars* tensors) {
    if (call->skip) return;
    const Chunk c = chunk_at(t, gridDim.x - 1 - blockIdx.x, kUpdateChunk);
    const TensorScalars s = tensors[t.first + c.tensor];
    const float scale = call->scale;
    const int dt = t.dtype[c.tensor];
    if (dt == kF32) update32<kF32, NT>(t, c, h, s, scale);
    else if (dt == kBF16) update32<kBF16, NT>(t, c, h, s, scale);
    else update32<kF16, NT>(t, c, h, s, scale);
}

constexpr int kTopM = 127, kTopV = 255, kNanM = 0x80;
constexpr int kFinite = 0x7F7;  // bits >> 20 of the largest finite number

__device__ __forceinline__ float decode_m(uint32_t code, int base) {
    if (code == kNanM) return __uint_as_float(0x7FC00000u);
    const uint32_t c = code & 127;
    return __uint_as_float((c ? uint32_t(base + int(c)) << 20 : 0u) | (code & 128) << 24);
}
__device__ __forceinline__ float decode_v(uint32_t code, int base) {
    return __uint_as_float(code ? uint32_t(base + int(code)) << 20 : 0u);
}
// `dither`: 16 bits, added centred below the mantissa bits that are kept.
__device__ __forceinline__ uint32_t encode_m(float m, int base, uint32_t dither) {
    const uint32_t bits = __float_as_uint(m), mag = bits & 0x7FFFFFFFu;
    uint32_t c;
    if (int(mag >> 20) <= base) {  // below the smallest code: that one, or zero, by chance
        const float least = __uint_as_float(uint32_t(base + 1) << 20);
        c = __uint_as_float(mag) * 65536.0f > (float(dither) + 0.5f) * least;
    } else {
        c = ((mag + (dither << 4) + 8) >> 20) - base;
    }
    return c ? c | (bits >> 24 & 128) : 0;
}
// `top`: the largest code of a finite number.
__device__ __forceinline__ uint32_t encode_v(float v, int base, int top, uint32_t dither) {
    const uint32_t bits = __float_as_uint(v);
    const int c = int((bits + (dither << 4) + 8) >> 20) - base;
    return bits == 0 ? 0 : uint32_t(min(max(c, 1), top));
}
__device__ __forceinline__ int base_of(uint32_t largest, int top) { return max(int(largest >> 20) + 1 - top, 0); }

__device__ __forceinline__ uint32_t max_partner(uint32_t v, int partner) { return max(v, uint32_t(partner)); }
// On every lane.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = max_partner(v, __builtin_amdgcn_update_dpp(0, int(v), 0x140, 0xf, 0xf, false));
    v = max_partner(v, __builtin_amdgcn_update_dpp(0, int(v), 0x141, 0xf, 0xf, false));
    v = max_partner(v, __builtin_amdgcn_update_dpp(0, int(v), 0x1b, 0xf, 0xf, false));
    v = max_partner(v, __builtin_amdgcn_update_dpp(0, int(v), 0xb1, 0xf, 0xf, false));
    auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(r[0], r[1]);
    r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max(r[0], r[1]);
}

__device__ __forceinline__ bool finite_bits(uint32_t magnitude) { return magnitude < 0x7F800000u; }

// A wavefront takes a block of 256 elements, four to a lane, and two blocks at a time.
template <int DT, bool NT>
__device__ __forceinline__ void update8(const AdamwTable& t, const Chunk& c, const Hyper& h, const TensorScalars& s,
                                        float scale) {
    constexpr int U = kUpdateVectors;
    const int lane = threadIdx.x & 63;
    const void* gs = t.g[c.tensor];
    void* ps = t.p[c.tensor];
    uint8_t *ms = static_cast<uint8_t*>(t.m[c.tensor]), *vs = static_cast<uint8_t*>(t.v[c.tensor]);
    Bases* bs = reinterpret_cast<Bases*>(t.bases[c.tensor]);
    const int64_t b = c.begin + (threadIdx.x >> 6) * kBlock;
    float p[U][4], g[U][4];
    uint32_t cm[U], cv[U], base[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t at = b + u * 4 * kBlock, e = at + lane * 4;
        load4<DT, NT>(gs, e, c.end, g[u]);
        load4<DT, NT>(ps, e, c.end, p[u]);
        cm[u] = load_codes(ms, e, c.end);
        cv[u] = load_codes(vs, e, c.end);
        base[u] = at < c.end ? bs[at / kBlock] : 0;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t at = b + u * 4 * kBlock, e = at + lane * 4;
        if (at >= c.end) break;
        const int bm = int16_t(base[u]), bv = int16_t(base[u] >> 16);
        Moments a[4];
        bool finite[4];
        uint32_t top_m = 0, top_v = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {  // past the end the codes and the gradient are 0, and so are the moments
            a[k] = moments(h, decode_m(cm[u] >> 8 * k & 255, bm), decode_v(cv[u] >> 8 * k & 255, bv),
                           g[u][k] * scale);
            p[u][k] = updated_fast(h, s, p[u][k], a[k]);
            const uint32_t um = __float_as_uint(a[k].m) & 0x7FFFFFFFu, uv = __float_as_uint(a[k].v);
            finite[k] = finite_bits(um) && finite_bits(uv);
            top_m = max(top_m, finite[k] ? um : 0);
            top_v = max(top_v, finite[k] ? uv : 0);
        }
        store4<DT, NT>(ps, e, c.end, p[u]);
        const int nm = base_of(wave_max(top_m), kTopM), nv = base_of(wave_max(top_v), kTopV);
        const int most_v = min(kTopV, kFinite - nv);  // (a finite v has an m far below the largest number)
        uint32_t om = 0, ov = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t r = mix(s.key + uint32_t(e + k) * 0x9E3779B1u);
            om |= (finite[k] ? encode_m(a[k].m, nm, r & 0xFFFF) : kNanM) << 8 * k;
            ov |= (finite[k] ? encode_v(a[k].v, nv, most_v, r >> 16) : kTopV) << 8 * k;
        }
        store_codes(ms, e, c.end, om);
        store_codes(vs, e, c.end, ov);
        if (lane == 0) bs[at / kBlock] = uint32_t(nm) | uint32_t(nv) << 16;
    }
}

template <bool NT>
__global__ __launch_bounds__(256) void k_adamw8(const AdamwTable t, const Hyper h, const CallScalars* call,
                                                const TensorScalars* tensors) {
    if (call->skip) return;
    const Chunk c = chunk_at(t, gridDim.x - 1 - blockIdx.x, kUpdateChunk);
    const TensorScalars s = tensors[t.first + c.tensor];
    const float scale = call->scale;
    const int dt = t.dtype[c.tensor];
    if (dt == kF32) update8<kF32, NT>(t, c, h, s, scale);
    else if (dt == kBF16) update8<kBF16, NT>(t, c, h, s, scale);
    else update8<kF16, NT>(t, c, h, s, scale);
}

// The moments that 8-bit states stand for: t.p and t.g receive m and v in float32.
template <bool NT>
__global__ __launch_bounds__(256) void k_adamw8_moments(const AdamwTable t) {
    constexpr int U = kUpdateVectors;
    const Chunk c = chunk_at(t, blockIdx.x, kUpdateChunk);
    const uint8_t *ms = static_cast<const uint8_t*>(t.m[c.tensor]), *vs = static_cast<const uint8_t*>(t.v[c.tensor]);
    const Bases* bs = reinterpret_cast<const Bases*>(t.bases[c.tensor]);
    void *mo = t.p[c.tensor], *vo = const_cast<void*>(t.g[c.tensor]);
    const int64_t b = c.begin + threadIdx.x * 4;
    uint32_t cm[U], cv[U], base[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t e = b + u * 1024;
        cm[u] = load_codes(ms, e, c.end);
        cv[u] = load_codes(vs, e, c.end);
        base[u] = e < c.end ? bs[e / kBlock] : 0;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float m[4], v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            m[k] = decode_m(cm[u] >> 8 * k & 255, int16_t(base[u]));
            v[k] = decode_v(cv[u] >> 8 * k & 255, int16_t(base[u] >> 16));
        }
        store4<kF32, NT>(mo, b + u * 1024, c.end, m);
        store4<kF32, NT>(vo, b + u * 1024, c.end, v);
    }
}

static int64_t total_of(const int64_t* numel, int64_t count) {
    int64_t total = 0;
    for (int64_t i = 0; i < count; ++i) total += std::max<int64_t>(numel[i], 0);
    return total;
}
// Partial sums of the norm.
static int64_t norm_chunks(const int64_t* numel, int64_t count) {
    const int chunk = norm_chunk(total_of(numel, count));
    int64_t chunks = 0;
    for (int64_t i = 0; i < count; ++i) chunks += ceil_div(std::max<int64_t>(numel[i], 0), chunk);
    return chunks;
}

// The first tensor of the launch whose last one is hi - 1: as many as a table holds and a grid takes.
static int64_t table_start(const int64_t* numel, int64_t hi) {
    int64_t lo = hi, chunks = 0;
    while (lo > 0 && hi - lo < kTensors) {
        chunks += ceil_div(numel[lo - 1], kUpdateChunk);
        if (lo < hi && chunks > kMostChunks) break;
        --lo;
    }
    return lo;
}

static int check_tensors(const char* what, int64_t count, const int64_t* numel, const int32_t* dtype) {
    MNX_REQUIRE(count >= 0 && count <= (1 << 30) && (count == 0 || numel), "%s: 0 to 2^30 tensors with their sizes",
                what);
    for (int64_t i = 0; i < count; ++i) {
        MNX_REQUIRE(numel[i] >= 0 && numel[i] <= MNX_OPTIM_MAX_ELEMENTS, "%s: tensor %lld has %lld elements", what,
                    (long long)i, (long long)numel[i]);
        MNX_REQUIRE(!dtype || elem_valid(dtype[i]), "%s: tensor %lld has an unknown element type", what, (long long)i);
    }
    return MNX_OK;
}

// Sums of squares of every chunk; `partial` has norm_chunks() places.
static int launch_sumsq(const void* const* grads, const int64_t* numel, const int32_t* dtype, int64_t count,
                        double* partial, mnx_stream_t stream) {
    NormTable t;
    t.count = 0;
    t.chunk = norm_chunk(total_of(numel, count));
    t.out = 0;
    uint32_t chunks = 0;
    auto flush = [&]() -> int {
        if (!t.count) return MNX_OK;
        t.start[t.count] = chunks;
        k_sumsq<<<chunks, 256, 0, stream>>>(t, partial);
        MNX_CHECK_LAUNCH();
        t.out += chunks;
        t.count = 0;
        chunks = 0;
        return MNX_OK;
    };
    for (int64_t i = 0; i < count; ++i) {
        if (!numel[i]) continue;
        MNX_REQUIRE(grads[i], "gradient norm: tensor %lld is null", (long long)i);
        const int64_t c = ceil_div(numel[i], t.chunk);
        if (t.count == kNormTensors || chunks + c > kMostChunks)
            if (int rc = flush()) return rc;
        t.g[t.count] = grads[i];
        t.n[t.count] = numel[i];
        t.dtype[t.count] = uint8_t(dtype[i]);
        t.start[t.count++] = chunks;
        chunks += uint32_t(c);
    }
    return flush();
}

}  // namespace mnx

using namespace mnx;

extern "C" {

size_t mnx_grad_norm_workspace_bytes(const int64_t* numel, int64_t count) {
    return size_t(std::max<int64_t>(count > 0 && numel ? norm_chunks(numel, count) : 0, 1)) * sizeof(double);
}

int mnx_grad_norm(const void* const* grads, const int64_t* numel, const int32_t* dtype, int64_t count, float* norm,
                  void* workspace, size_t workspace_bytes, mnx_stream_t stream) {
    clear_error();
    if (int rc = check_tensors("gradient norm", count, numel, dtype)) return rc;
    MNX_REQUIRE(norm && (count == 0 || (grads && dtype)), "gradient norm: null pointer");
    if (!workspace || workspace_bytes < mnx_grad_norm_workspace_bytes(numel, count))
        return set_error(MNX_ERR_WORKSPACE, "gradient norm: workspace too small");
    double* partial = static_cast<double*>(workspace);
    if (int rc = launch_sumsq(grads, numel, dtype, count, partial, stream)) return rc;
    k_norm<<<1, 1024, 0, stream>>>(partial, norm_chunks(numel, count), norm);
    MNX_CHECK_LAUNCH();
    return MNX_OK;
}

size_t mnx_adamw_workspace_bytes(const int64_t* numel, int64_t count) {
    Workspace ws{nullptr, 0};
    ws.take<CallScalars>(1);
    ws.take<TensorScalars>(size_t(std::max<int64_t>(count, 1)));
    ws.take<char>(mnx_grad_norm_workspace_bytes(numel, count));
    return ws.used;
}

int mnx_adamw_step(const mnx_adamw_args* args, mnx_stream_t stream) {
    clear_error();
    MNX_REQUIRE(args, "adamw: null arguments");
    const mnx_adamw_args& a = *args;
    if (int rc = check_tensors("adamw", a.count, a.numel, a.dtype)) return rc;
    MNX_REQUIRE(a.state_bits == 8 || a.state_bits == 32, "adamw: state_bits 8 or 32, got %d", a.state_bits);
    const bool eight = a.state_bits == 8;
    if (a.count == 0 && !a.norm_out) return MNX_OK;
    MNX_REQUIRE(a.count == 0 || (a.params && a.grads && a.exp_avgs && a.exp_avg_sqs && a.steps && a.dtype &&
                                 (!eight || a.bases)),
                "adamw: null pointer");
    MNX_REQUIRE(a.beta1 >= 0 && a.beta1 < 1 && a.beta2 >= 0 && a.beta2 < 1 && a.eps >= 0,
                "adamw: 0 <= beta < 1, eps >= 0");
    for (int64_t i = 0; i < a.count; ++i)
        MNX_REQUIRE(a.steps[i] && (!a.numel[i] || (a.params[i] && a.grads[i] && a.exp_avgs[i] && a.exp_avg_sqs[i] &&
                                                   (!eight || a.bases[i]))),
                    "adamw: tensor %lld has a null pointer", (long long)i);
    Workspace ws{static_cast<char*>(a.workspace), a.workspace_bytes};
    CallScalars* call = ws.take<CallScalars>(1);
    TensorScalars* scalars = ws.take<TensorScalars>(size_t(std::max<int64_t>(a.count, 1)));
    const int64_t chunks = norm_chunks(a.numel, a.count);
    double* partial = ws.take<double>(size_t(std::max<int64_t>(chunks, 1)));
    if (!a.workspace || !ws.fits()) return set_error(MNX_ERR_WORKSPACE, "adamw: workspace too small");

    const bool own_norm = (a.max_norm >= 0 || a.skip_nonfinite || a.norm_out) && !a.norm_in;
    if (own_norm)
        if (int rc = launch_sumsq(a.grads, a.numel, a.dtype, a.count, partial, stream)) return rc;
    StepTable st;
    for (int64_t at = 0; at == 0 || at < a.count; at += kStepTensors) {
        st.first = int(at);
        st.count = int(std::min<int64_t>(kStepTensors, a.count - at));
        for (int i = 0; i < st.count; ++i) st.step[i] = a.steps[at + i];
        k_adamw_prepare<<<1, 1024, 0, stream>>>(st, own_norm ? partial : nullptr, chunks, a.norm_in, a.norm_out,
                                               a.max_norm, a.skip_nonfinite, a.maximize, a.lr, a.lr_device, a.beta1,
                                               a.beta2, a.weight_decay, a.seed, call, scalars);
        MNX_CHECK_LAUNCH();
    }
    // An eps below the smallest normal number counts as that one: its only use is beside a second moment of zero, and
    // the reciprocal's instruction takes no subnormals.
    const float eps = a.eps > 0 ? std::max(float(a.eps), 0x1p-126f) : 0.0f;
    const Hyper h{float(a.beta1), float(1 - a.beta1), float(a.beta2), float(1 - a.beta2), eps};
    int64_t bytes = 0;
    for (int64_t i = 0; i < a.count; ++i) bytes += a.numel[i] * (3 * elem_bytes(a.dtype[i]) + (eight ? 4 : 16));
    const auto kernel = bytes > kCacheBytes ? (eight ? k_adamw8<true> : k_adamw<true>)
                                            : (eight ? k_adamw8<false> : k_adamw<false>);
    for (int64_t hi = a.count, lo; hi > 0; hi = lo) {  // the last tensors first
        AdamwTable t;
        lo = table_start(a.numel, hi);
        t.first = int(lo);
        t.count = int(hi - lo);
        uint32_t c = 0;
        for (int i = 0; i < t.count; ++i) {
            t.p[i] = a.params[lo + i];
            t.g[i] = a.grads[lo + i];
            t.m[i] = a.exp_avgs[lo + i];
            t.v[i] = a.exp_avg_sqs[lo + i];
            t.bases[i] = eight ? a.bases[lo + i] : nullptr;
            t.n[i] = a.numel[lo + i];
            t.dtype[i] = uint8_t(a.dtype[lo + i]);
            t.start[i] = c;
            c += uint32_t(ceil_div(t.n[i], kUpdateChunk));
        }
        t.start[t.count] = c;
        if (!c) continue;
        kernel<<<c, 256, 0, stream>>>(t, h, call, scalars);
        MNX_CHECK_LAUNCH();
    }
    return MNX_OK;
}

int mnx_adamw8_moments(const void* const* exp_avgs, const void* const* exp_avg_sqs, int16_t* const* bases,
                       const int64_t* numel, int64_t count, float* const* out_avgs, float* const* out_avg_sqs,
                       mnx_stream_t stream) {
    clear_error();
    if (int rc = check_tensors("adamw8 moments", count, numel, nullptr)) return rc;
    MNX_REQUIRE(count == 0 || (exp_avgs && exp_avg_sqs && bases && out_avgs && out_avg_sqs),
                "adamw8 moments: null pointer");
    const auto kernel = total_of(numel, count) * 10 > kCacheBytes ? k_adamw8_moments<true> : k_adamw8_moments<false>;
    for (int64_t hi = count, lo; hi > 0; hi = lo) {
        AdamwTable t;
        lo = table_start(numel, hi);
        t.first = int(lo);
        t.count = int(hi - lo);
        uint32_t c = 0;
        for (int i = 0; i < t.count; ++i) {
            const int64_t k = lo + i;
            MNX_REQUIRE(!numel[k] || (exp_avgs[k] && exp_avg_sqs[k] && bases[k] && out_avgs[k] && out_avg_sqs[k]),
                        "adamw8 moments: tensor %lld has a null pointer", (long long)k);
            t.p[i] = out_avgs[k];
            t.g[i] = out_avg_sqs[k];
            t.m[i] = const_cast<void*>(exp_avgs[k]);
            t.v[i] = const_cast<void*>(exp_avg_sqs[k]);
            t.bases[i] = bases[k];
            t.n[i] = numel[k];
            t.dtype[i] = kF32;
            t.start[i] = c;
            c += uint32_t(ceil_div(t.n[i], kUpdateChunk));
        }
        t.start[t.count] = c;
        if (!c) continue;
        kernel<<<c, 256, 0, stream>>>(t);
        MNX_CHECK_LAUNCH();
    }
    return MNX_OK;
}

}  // extern "C"
