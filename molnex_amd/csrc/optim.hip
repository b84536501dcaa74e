// AdamW over many tensors, with 32-bit or 8-bit states, and the 2-norm of many tensors.
//
//   g' = s g, s = min(1, max_norm / (norm + 1e-6)) (1 without a max_norm);  t += 1
//   m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g' g'
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// The tensors' addresses travel in the kernels' arguments (a table of up to kTensors entries a launch), so a call
// copies nothing to the device and can be captured in a graph; the step counts t, the norm and what follows from
// them stay on the device.  A workgroup takes a chunk of one tensor.
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
constexpr int kStepTensors = 480;  // tensors of one launch of the step counts
constexpr int kBlock = 256;        // elements of a block of 8-bit states
constexpr int kChunk = 8192;       // elements a workgroup takes

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
    int count;
    int64_t out;  // place of the first chunk's partial sum
};

struct StepTable {
    float* step[kStepTensors];
    int count, first;
};

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

// Sums over the workgroup of 256, valid on thread 0.
__device__ __forceinline__ double block_sum(double v) {
    __shared__ double part[4];
    for (int off = 32; off; off >>= 1) v += __shfl_xor(v, off);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (part[0] + part[1]) + (part[2] + part[3]);
    __syncthreads();
    return v;
}

// Squares are summed in float64: no overflow where the norm itself has none, and the same last bits whatever the
// order of the chunks.
__global__ __launch_bounds__(256) void k_sumsq(const NormTable t, double* partial) {
    const int i = find_tensor(t.start, t.count, blockIdx.x);
    const int64_t begin = int64_t(blockIdx.x - t.start[i]) * kChunk, end = min(t.n[i], begin + kChunk);
    double s = 0;
    for (int64_t e = begin + threadIdx.x; e < end; e += 256) {
        const double g = load_elem(t.g[i], e, t.dtype[i]);
        s += g * g;
    }
    s = block_sum(s);
    if (threadIdx.x == 0) partial[t.out + blockIdx.x] = s;
}

__device__ __forceinline__ double sum_partial(const double* partial, int64_t chunks) {
    double s = 0;
    for (int64_t i = threadIdx.x; i < chunks; i += 256) s += partial[i];
    return block_sum(s);
}

__global__ __launch_bounds__(256) void k_norm(const double* partial, int64_t chunks, float* norm) {
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

// The step counts and everything that the update takes from them and from the norm, in float64.
__global__ __launch_bounds__(256) void k_adamw_prepare(const StepTable t, const double* partial, int64_t chunks,
                                                       const float* norm_in, float* norm_out, double max_norm,
                                                       int skip_nonfinite, int maximize, double lr, const float* lr_dev,
                                                       double b1, double b2, double wd, uint32_t seed,
                                                       CallScalars* call, TensorScalars* tensors) {
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
    if (skip) return;
    if (lr_dev) lr = *lr_dev;
    for (int i = threadIdx.x; i < t.count; i += 256) {
        const float step = *t.step[i] + 1.0f;
        *t.step[i] = step;
        TensorScalars s;
        s.size = float(lr / (1 - pow(b1, double(step))));
        s.inv_root = float(1 / sqrt(1 - pow(b2, double(step))));
        s.decay = float(1 - lr * wd);
        s.key = mix(mix(seed * 0x3C6EF373u + uint32_t(t.first + i) * 0xA54FF53Bu) + uint32_t(step) * 0x510E527Fu);
        tensors[t.first + i] = s;
    }
}

struct Moments {
    float m, v;
};

__device__ __forceinline__ Moments moments(const Hyper& h, float m, float v, float g) {
    return {m * h.b1 + g * h.w1, v * h.b2 + (g * g) * h.w2};
}
__device__ __forceinline__ float updated(const Hyper& h, const TensorScalars& s, float p, const Moments& a) {
    return p * s.decay - s.size * a.m / (sqrtf(a.v) * s.inv_root + h.eps);
}

__global__ __launch_bounds__(256) void k_adamw(const AdamwTable t, const Hyper h, const CallScalars* call,
                                               const TensorScalars* tensors) {
    if (call->skip) return;
    const int i = find_tensor(t.start, t.count, blockIdx.x);
    const int64_t begin = int64_t(blockIdx.x - t.start[i]) * kChunk, end = min(t.n[i], begin + kChunk);
    const TensorScalars s = tensors[t.first + i];
    const float scale = call->scale;
    float *m = static_cast<float*>(t.m[i]), *v = static_cast<float*>(t.v[i]);
    for (int64_t e = begin + threadIdx.x; e < end; e += 256) {
        const Moments a = moments(h, m[e], v[e], load_elem(t.g[i], e, t.dtype[i]) * scale);
        store_elem(t.p[i], e, t.dtype[i], updated(h, s, load_elem(t.p[i], e, t.dtype[i]), a));
        m[e] = a.m;
        v[e] = a.v;
    }
}

constexpr int kTopM = 127, kTopV = 255, kNanM = 0x80;

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
__device__ __forceinline__ uint32_t encode_v(float v, int base, uint32_t dither) {
    const uint32_t bits = __float_as_uint(v);
    const int c = int((bits + (dither << 4) + 8) >> 20) - base;
    return bits == 0 ? 0 : uint32_t(min(max(c, 1), kTopV));
}
__device__ __forceinline__ int base_of(uint32_t largest, int top) { return max(int(largest >> 20) + 1 - top, 0); }

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    for (int off = 32; off; off >>= 1) v = max(v, uint32_t(__shfl_xor(int(v), off)));
    return v;
}

// A wavefront takes a block of 256 elements, four to a lane.
__global__ __launch_bounds__(256) void k_adamw8(const AdamwTable t, const Hyper h, const CallScalars* call,
                                                const TensorScalars* tensors) {
    if (call->skip) return;
    const int i = find_tensor(t.start, t.count, blockIdx.x);
    const int64_t begin = int64_t(blockIdx.x - t.start[i]) * kChunk, n = t.n[i], end = min(n, begin + kChunk);
    const TensorScalars s = tensors[t.first + i];
    const float scale = call->scale;
    uint8_t *cm = static_cast<uint8_t*>(t.m[i]), *cv = static_cast<uint8_t*>(t.v[i]);
    const int lane = threadIdx.x & 63;
    for (int64_t b = begin + (threadIdx.x >> 6) * kBlock; b < end; b += 4 * kBlock) {
        int16_t* bases = t.bases[i] + b / kBlock * 2;
        const int bm = bases[0], bv = bases[1];
        Moments a[4];
        uint32_t top_m = 0, top_v = 0;
        for (int k = 0; k < 4; ++k) {
            const int64_t e = b + lane * 4 + k;
            a[k] = {0, 0};
            if (e >= n) continue;
            a[k] = moments(h, decode_m(cm[e], bm), decode_v(cv[e], bv), load_elem(t.g[i], e, t.dtype[i]) * scale);
            store_elem(t.p[i], e, t.dtype[i], updated(h, s, load_elem(t.p[i], e, t.dtype[i]), a[k]));
            const uint32_t um = __float_as_uint(a[k].m) & 0x7FFFFFFFu, uv = __float_as_uint(a[k].v);
            if (um < 0x7F800000u && uv < 0x7F800000u) {
                top_m = max(top_m, um);
                top_v = max(top_v, uv);
            }
        }
        const int nm = base_of(wave_max(top_m), kTopM), nv = base_of(wave_max(top_v), kTopV);
        for (int k = 0; k < 4; ++k) {
            const int64_t e = b + lane * 4 + k;
            if (e >= n) continue;
            const uint32_t r = mix(s.key + uint32_t(e) * 0x9E3779B1u);
            const bool finite = (__float_as_uint(a[k].m) & 0x7FFFFFFFu) < 0x7F800000u &&
                                __float_as_uint(a[k].v) < 0x7F800000u;
            cm[e] = finite ? encode_m(a[k].m, nm, r & 0xFFFF) : kNanM;
            cv[e] = finite ? encode_v(a[k].v, nv, r >> 16) : kTopV;
        }
        if (lane == 0) bases[0] = int16_t(nm), bases[1] = int16_t(nv);
    }
}

// The moments that 8-bit states stand for: t.p and t.g receive m and v in float32.
__global__ __launch_bounds__(256) void k_adamw8_moments(const AdamwTable t) {
    const int i = find_tensor(t.start, t.count, blockIdx.x);
    const int64_t begin = int64_t(blockIdx.x - t.start[i]) * kChunk, end = min(t.n[i], begin + kChunk);
    const uint8_t *cm = static_cast<const uint8_t*>(t.m[i]), *cv = static_cast<const uint8_t*>(t.v[i]);
    float *m = static_cast<float*>(t.p[i]), *v = static_cast<float*>(const_cast<void*>(t.g[i]));
    for (int64_t e = begin + threadIdx.x; e < end; e += 256) {
        const int16_t* bases = t.bases[i] + e / kBlock * 2;
        m[e] = decode_m(cm[e], bases[0]);
        v[e] = decode_v(cv[e], bases[1]);
    }
}

static int64_t chunks_of(const int64_t* numel, int64_t count) {
    int64_t chunks = 0;
    for (int64_t i = 0; i < count; ++i) chunks += ceil_div(std::max<int64_t>(numel[i], 0), kChunk);
    return chunks;
}

static int check_tensors(const char* what, int64_t count, const int64_t* numel, const int32_t* dtype) {
    MNX_REQUIRE(count >= 0 && (count == 0 || numel), "%s: no tensors' sizes", what);
    for (int64_t i = 0; i < count; ++i) {
        MNX_REQUIRE(numel[i] >= 0 && numel[i] <= MNX_OPTIM_MAX_ELEMENTS, "%s: tensor %lld has %lld elements", what,
                    (long long)i, (long long)numel[i]);
        MNX_REQUIRE(!dtype || elem_valid(dtype[i]), "%s: tensor %lld has an unknown element type", what, (long long)i);
    }
    return MNX_OK;
}

// Sums of squares of every chunk; `partial` has chunks_of() places.
static int launch_sumsq(const void* const* grads, const int64_t* numel, const int32_t* dtype, int64_t count,
                        double* partial, mnx_stream_t stream) {
    NormTable t;
    t.count = 0;
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
        const int64_t c = ceil_div(numel[i], kChunk);
        if (t.count == kNormTensors || chunks + c > (1u << 23))
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
    return size_t(std::max<int64_t>(count > 0 && numel ? chunks_of(numel, count) : 0, 1)) * sizeof(double);
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
    k_norm<<<1, 256, 0, stream>>>(partial, chunks_of(numel, count), norm);
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
    MNX_REQUIRE(a.beta1 >= 0 && a.beta1 < 1 && a.beta2 >= 0 && a.beta2 < 1 && a.eps >= 0, "adamw: 0 <= beta < 1, eps >= 0");
    for (int64_t i = 0; i < a.count; ++i)
        MNX_REQUIRE(a.steps[i] && (!a.numel[i] || (a.params[i] && a.grads[i] && a.exp_avgs[i] && a.exp_avg_sqs[i] &&
                                                   (!eight || a.bases[i]))),
                    "adamw: tensor %lld has a null pointer", (long long)i);
    Workspace ws{static_cast<char*>(a.workspace), a.workspace_bytes};
    CallScalars* call = ws.take<CallScalars>(1);
    TensorScalars* scalars = ws.take<TensorScalars>(size_t(std::max<int64_t>(a.count, 1)));
    const int64_t chunks = chunks_of(a.numel, a.count);
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
        k_adamw_prepare<<<1, 256, 0, stream>>>(st, own_norm ? partial : nullptr, chunks, a.norm_in, a.norm_out,
                                               a.max_norm, a.skip_nonfinite, a.maximize, a.lr, a.lr_device, a.beta1,
                                               a.beta2, a.weight_decay, a.seed, call, scalars);
        MNX_CHECK_LAUNCH();
    }
    const Hyper h{float(a.beta1), float(1 - a.beta1), float(a.beta2), float(1 - a.beta2), float(a.eps)};
    AdamwTable t;
    for (int64_t at = 0; at < a.count; at += kTensors) {
        t.first = int(at);
        t.count = int(std::min<int64_t>(kTensors, a.count - at));
        int64_t c = 0;
        for (int i = 0; i < t.count; ++i) {
            t.p[i] = a.params[at + i];
            t.g[i] = a.grads[at + i];
            t.m[i] = a.exp_avgs[at + i];
            t.v[i] = a.exp_avg_sqs[at + i];
            t.bases[i] = eight ? a.bases[at + i] : nullptr;
            t.n[i] = a.numel[at + i];
            t.dtype[i] = uint8_t(a.dtype[at + i]);
            t.start[i] = uint32_t(c);
            c += ceil_div(t.n[i], kChunk);
        }
        t.start[t.count] = uint32_t(c);
        if (!c) continue;
        if (eight) k_adamw8<<<uint32_t(c), 256, 0, stream>>>(t, h, call, scalars);
        else k_adamw<<<uint32_t(c), 256, 0, stream>>>(t, h, call, scalars);
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
    AdamwTable t;
    for (int64_t at = 0; at < count; at += kTensors) {
        t.first = int(at);
        t.count = int(std::min<int64_t>(kTensors, count - at));
        int64_t c = 0;
        for (int i = 0; i < t.count; ++i) {
            const int64_t k = at + i;
            MNX_REQUIRE(!numel[k] || (exp_avgs[k] && exp_avg_sqs[k] && bases[k] && out_avgs[k] && out_avg_sqs[k]),
                        "adamw8 moments: tensor %lld has a null pointer", (long long)k);
            t.p[i] = out_avgs[k];
            t.g[i] = out_avg_sqs[k];
            t.m[i] = const_cast<void*>(exp_avgs[k]);
            t.v[i] = const_cast<void*>(exp_avg_sqs[k]);
            t.bases[i] = bases[k];
            t.n[i] = numel[k];
            t.dtype[i] = kF32;
            t.start[i] = uint32_t(c);
            c += ceil_div(t.n[i], kChunk);
        }
        t.start[t.count] = uint32_t(c);
        if (!c) continue;
        k_adamw8_moments<<<uint32_t(c), 256, 0, stream>>>(t);
        MNX_CHECK_LAUNCH();
    }
    return MNX_OK;
}

}  // extern "C"
