// Adam / AdamW over many tensors in a few launches, moments in 32 bits or in 8, gradient clipping by the global norm.
//
// Mathematics, per element (t: the tensor's step counter after this step):
//   c = min(1, max_norm / (|g| + 1e-6))                  |g| over all gradients, summed in 64 bits
//   g = c g (+ wd p: weight decay in the gradient)        m = b1 m + (1 - b1) g        v = b2 v + (1 - b2) g^2
//   p = p (- lr wd p: decoupled decay) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// Every operation is rounded on its own to 32 bits (this file is built without contraction), so a step is the same
// numbers as the same operations in elementary tensor code.
//
// What bounds it: memory.  A 32-bit step reads 16 and writes 12 bytes per weight, an 8-bit one 10 and 6; clipping reads
// the gradients once more.  The pointers travel in the kernel arguments (at most AZ_OPTIM_TABLE tensors a launch):
// nothing is uploaded, so the step can be captured, and tensors may move between steps.
#include <math.h>

#include "train_common.h"

namespace az {

constexpr int OPT_THREADS = 256;
constexpr int OPT_CHUNK = AZ_OPTIM_CHUNK;          // elements of one tensor that one workgroup takes
constexpr int OPT_BLOCK = AZ_OPTIM_PAD;            // elements that share a scale: one wavefront x 4
constexpr int OPT_TABLE = 136;                     // 28 bytes each: 3.8 KB of the 4 KB of kernel arguments
constexpr int OPT_SLOTS = 960;
static_assert(OPT_CHUNK % (OPT_THREADS * 4) == 0 && OPT_BLOCK == 256, "a wavefront covers one block of a moment");

struct OptTable {
    uint64_t grad[OPT_TABLE];
    uint64_t param[OPT_TABLE];
    uint32_t first[OPT_TABLE];      // first workgroup of the tensor in this launch
    uint32_t offset[OPT_TABLE];     // its place in the moments, in units of OPT_BLOCK
    uint32_t slot_tail[OPT_TABLE];  // step counter (20 bits) | elements of the last chunk - 1 (12 bits)
    uint32_t count, chunks;
};

struct SlotList {
    uint32_t slot[OPT_SLOTS];
};

struct StepFactors {                // per tensor, from its step counter
    float step_size, inv_root_bias2;
    uint32_t key;
};

struct OptHyper {
    double lr, beta1, beta2, max_norm;
    const double* partials;
    uint32_t n_partials;
    float* norm;                    // |g| out (may be null)
    float* coef;                    // c out
    float* steps;
    StepFactors* factors;
    uint32_t seed_key;
};

struct AdamParams {
    float beta1, one_beta1, beta2, one_beta2, eps, decay;   // decay: wd, or 1 - lr wd
    int decoupled;
    const float* coef;
    const StepFactors* factors;
    void *m, *v;
    float *m_scale, *v_scale;
};

// The tensor that workgroup b works on.  Every lane compares its part of `first`: one round trip instead of the
// eight of a search by halves.
__device__ inline uint32_t find_tensor(const OptTable& t, uint32_t b) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t n = 0;
#pragma unroll
    for (uint32_t k = 0; k < OPT_TABLE; k += 64) {
        const uint32_t i = k + lane;
        const bool at_or_before = i < t.count && t.first[i < OPT_TABLE ? i : 0] <= b;
        n += __popcll(__ballot(at_or_before));
    }
    return __builtin_amdgcn_readfirstlane(n - 1);
}

struct Chunk {
    uint32_t tensor, index, n;     // which tensor, which chunk of it, its elements
};

__device__ inline Chunk find_chunk(const OptTable& t, uint32_t b) {
    Chunk c;
    c.tensor = find_tensor(t, b);
    c.index = b - t.first[c.tensor];
    const uint32_t end = c.tensor + 1 < t.count ? t.first[c.tensor + 1] : t.chunks;
    c.n = b + 1 == end ? (t.slot_tail[c.tensor] >> 20) + 1 : OPT_CHUNK;
    return c;
}

// Sum of squares of a chunk in 64 bits (the products are exact there): the norm of 8 M gradients whose sizes lie decades
// apart, and a clipping factor that does not depend on the order of the sum.
__global__ __launch_bounds__(OPT_THREADS) void k_grad_sumsq(const OptTable t, double* partials) {
    const Chunk c = find_chunk(t, blockIdx.x);
    const float* g = (const float*)t.grad[c.tensor] + (size_t)c.index * OPT_CHUNK;
    double s = 0.0;
#pragma unroll
    for (int it = 0; it < OPT_CHUNK / (OPT_THREADS * 4); ++it) {
        const int i = it * OPT_THREADS * 4 + threadIdx.x * 4;
        const f32x4 v = load_pack(g + i, (int)c.n - i);
#pragma unroll
        for (int k = 0; k < 4; ++k) s += (double)v[k] * (double)v[k];
    }
    for (int off = 32; off; off >>= 1) s += __shfl_xor(s, off);
    __shared__ double part[OPT_THREADS / 64];
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < OPT_THREADS / 64; ++w) s += part[w];
        partials[blockIdx.x] = s;
    }
}

// One workgroup: the norm and the clipping factor from the partial sums (in a fixed order), and the tensors' step
// counters with what follows from them.
__global__ __launch_bounds__(1024) void k_adam_begin(const SlotList l, uint32_t count, OptHyper h) {
    if (h.coef) {
        double s = 0.0;
        for (uint32_t i = threadIdx.x; i < h.n_partials; i += 1024) s += h.partials[i];
        for (int off = 32; off; off >>= 1) s += __shfl_xor(s, off);
        __shared__ double part[16];
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < 16; ++w) s += part[w];
            const double norm = sqrt(s), c = h.max_norm / (norm + 1e-6);
            if (h.norm) *h.norm = (float)norm;
            *h.coef = (float)(c > 1.0 ? 1.0 : c);      // a NaN stays one
        }
    }
    for (uint32_t i = threadIdx.x; i < count; i += 1024) {
        const uint32_t slot = l.slot[i];
        const float t = h.steps[slot] + 1.f;
        h.steps[slot] = t;
        StepFactors f;
        f.step_size = (float)(h.lr / (1.0 - pow(h.beta1, (double)t)));
        f.inv_root_bias2 = 1.f / (float)sqrt(1.0 - pow(h.beta2, (double)t));
        f.key = h.seed_key + (uint32_t)t * 0x85EBCA6Bu;
        h.factors[slot] = f;
    }
}

// ---- moments in 8 bits -------------------------------------------------------------------------------------------
// 256 values share a power of two that puts their largest in (224, 448]; each is an e4m3 code times it: 3 bits of
// mantissa over 17 binades, both directions of the scaling exact.  m is held as itself, v as its root: the root is what
// the update divides by, and squaring 17 binades would lose the small ones.  A decaying average moves by less than half
// a code's step (6 %) per step, so rounding to nearest would freeze it: values are rounded at random, up with the
// probability of the way they have gone, which keeps the averages right.  A root that is not zero never becomes zero
// (the update would divide by eps alone).  What is not finite becomes the code of NaN.
__device__ inline float block_top(const f32x4 x) {
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float a = fabsf(x[k]);
        top = fmaxf(top, a <= 3.402823466e38f ? a : 0.f);
    }
    return lane_max<64>(top);
}

__device__ inline int scale_exponent(float top) {
    const uint32_t b = __float_as_uint(top);
    const int k = (int)(b >> 23) - 127 - 8 + ((b & 0x7FFFFFu) > 0x600000u);
    return k < -108 ? -108 : k;
}

__device__ inline float pow2(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }

__device__ inline uint32_t encode(float x, float inv_scale, uint32_t r16, bool keep) {
    const float y = fabsf(x) * inv_scale;
    const int e = (int)(__float_as_uint(y) >> 23) - 127, place = (e < -6 ? -6 : e) - 3;
    const float q = floorf(y * pow2(-place) + (float)r16 * (1.f / 65536.f));
    uint32_t code = ((uint32_t)(place + 9) << 3) + (uint32_t)q;
    if (keep && code == 0 && y > 0.f) code = 1;
    if (!(y <= 448.f)) code = 0x7F;
    return code | (__float_as_uint(x) >> 31 << 7);
}

__device__ inline f32x4 decode(uint32_t codes, float scale) {
    f32x4 r;
    r[0] = __builtin_amdgcn_cvt_f32_fp8(codes, 0) * scale;
    r[1] = __builtin_amdgcn_cvt_f32_fp8(codes, 1) * scale;
    r[2] = __builtin_amdgcn_cvt_f32_fp8(codes, 2) * scale;
    r[3] = __builtin_amdgcn_cvt_f32_fp8(codes, 3) * scale;
    return r;
}

__device__ inline uint32_t mix32(uint32_t z) {
    z = (z ^ (z >> 16)) * 0x7FEB352Du;
    z = (z ^ (z >> 15)) * 0x846CA68Bu;
    return z ^ (z >> 16);
}

template <int BITS>
__global__ __launch_bounds__(OPT_THREADS) void k_adam(const OptTable t, const AdamParams a) {
    const Chunk c = find_chunk(t, blockIdx.x);
    const float* gp = (const float*)t.grad[c.tensor] + (size_t)c.index * OPT_CHUNK;
    float* pp = (float*)t.param[c.tensor] + (size_t)c.index * OPT_CHUNK;
    const size_t at = (size_t)t.offset[c.tensor] * OPT_BLOCK + (size_t)c.index * OPT_CHUNK;   // place in the moments
    const StepFactors f = a.factors[t.slot_tail[c.tensor] & 0xFFFFFu];
    const float coef = a.coef ? *a.coef : 1.f;
#pragma unroll
    for (int it = 0; it < OPT_CHUNK / (OPT_THREADS * 4); ++it) {
        const int i = it * OPT_THREADS * 4 + threadIdx.x * 4, left = (int)c.n - i;
        if (left + (int)(threadIdx.x & 63) * 4 <= 0) break;             // the wavefront's whole block is past the end
        f32x4 p = load_pack((const float*)pp + i, left), g = load_pack(gp + i, left), m, v;
        // the moments' own places run on to a multiple of OPT_BLOCK: no tail there
        if (BITS == 32) {
            m = *(const f32x4*)((const float*)a.m + at + i);
            v = *(const f32x4*)((const float*)a.v + at + i);
        } else {
            m = decode(*(const uint32_t*)((const uint8_t*)a.m + at + i), a.m_scale[(at + i) / OPT_BLOCK]);
            v = decode(*(const uint32_t*)((const uint8_t*)a.v + at + i), a.v_scale[(at + i) / OPT_BLOCK]);
        }
        f32x4 root;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float gk = g[k], pk = p[k];
            if (a.coef) gk = gk * coef;
            if (a.decoupled) pk = pk * a.decay;
            else if (a.decay != 0.f) gk = gk + pk * a.decay;
            const float vk = BITS == 32 ? v[k] : v[k] * v[k];
            m[k] = m[k] * a.beta1 + gk * a.one_beta1;
            v[k] = vk * a.beta2 + gk * gk * a.one_beta2;
            root[k] = sqrtf(v[k]);
            p[k] = pk - m[k] / (root[k] * f.inv_root_bias2 + a.eps) * f.step_size;
        }
        store_pack(pp + i, p, left);
        if (BITS == 32) {
            *(f32x4*)((float*)a.m + at + i) = m;
            *(f32x4*)((float*)a.v + at + i) = v;
        } else {
            const int km = scale_exponent(block_top(m)), kv = scale_exponent(block_top(root));
            uint32_t cm = 0, cv = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t place = (uint32_t)(at + i + k), r = mix32(place + f.key);
                cm |= encode(m[k], pow2(-km), r & 0xFFFF, false) << (8 * k);
                cv |= encode(root[k], pow2(-kv), r >> 16, true) << (8 * k);
            }
            *(uint32_t*)((uint8_t*)a.m + at + i) = cm;
            *(uint32_t*)((uint8_t*)a.v + at + i) = cv;
            if ((threadIdx.x & 63) == 0) {
                a.m_scale[(at + i) / OPT_BLOCK] = pow2(km);
                a.v_scale[(at + i) / OPT_BLOCK] = pow2(kv);
            }
        }
    }
}

// Splits a list of tensors into launches and calls launch(table, chunks before it).
template <typename F>
static int for_tables(int32_t count, const uint64_t* params, const uint64_t* grads, const int64_t* sizes,
                      const int64_t* offsets, const int32_t* slots, F&& launch) {
    OptTable t;
    t.count = t.chunks = 0;
    int64_t before = 0;
    for (int32_t i = 0; i < count; ++i) {
        const int64_t n = sizes[i];
        AZ_CHECK_ARG(n >= 0 && n <= (int64_t(1) << 40), "tensor %d has %lld elements", i, (long long)n);
        if (n == 0) continue;
        AZ_CHECK_ARG(grads[i] && grads[i] % 4 == 0, "gradient %d is null or not aligned to 4 bytes", i);
        const int64_t chunks = (n + OPT_CHUNK - 1) / OPT_CHUNK;
        if (t.count == (uint32_t)OPT_TABLE || (t.count && t.chunks + chunks > 0x7FFFFFFF)) {
            const int rc = launch(t, before);
            if (rc != AZ_OK) return rc;
            before += t.chunks;
            t.count = t.chunks = 0;
        }
        t.grad[t.count] = grads[i];
        t.param[t.count] = params ? params[i] : 0;
        t.first[t.count] = t.chunks;
        t.offset[t.count] = offsets ? (uint32_t)(offsets[i] / OPT_BLOCK) : 0;
        t.slot_tail[t.count] = (slots ? (uint32_t)slots[i] : 0) | (uint32_t)(n - (chunks - 1) * OPT_CHUNK - 1) << 20;
        ++t.count;
        t.chunks += (uint32_t)chunks;
    }
    return t.count ? launch(t, before) : AZ_OK;
}

}  // namespace az

using namespace az;

extern "C" int az_grad_sumsq(int32_t count, const uint64_t* grads_host, const int64_t* sizes_host, double* partials_dev,
                             int64_t n_partials, void* stream) {
    AZ_CHECK_ARG(count >= 0 && (count == 0 || (grads_host && sizes_host)), "az_grad_sumsq: null table");
    int64_t need = 0;
    for (int32_t i = 0; i < count; ++i) need += sizes_host[i] > 0 ? (sizes_host[i] + OPT_CHUNK - 1) / OPT_CHUNK : 0;
    AZ_CHECK_ARG(n_partials >= need && (need == 0 || partials_dev), "az_grad_sumsq: %lld partial sums needed, room for %lld",
                 (long long)need, (long long)n_partials);
    return for_tables(count, nullptr, grads_host, sizes_host, nullptr, nullptr, [&](const OptTable& t, int64_t before) -> int {
        hipLaunchKernelGGL(k_grad_sumsq, dim3(t.chunks), dim3(OPT_THREADS), 0, (hipStream_t)stream, t, partials_dev + before);
        AZ_HIP(hipGetLastError());
        return AZ_OK;
    });
}

extern "C" int az_adam_step(const az_adam_config* cfg, int32_t count, const uint64_t* params_host, const uint64_t* grads_host,
                            const int64_t* sizes_host, const int64_t* offsets_host, const int32_t* slots_host, void* stream) {
    AZ_CHECK_ARG(cfg, "az_adam_step: null config");
    if (count == 0) return AZ_OK;
    AZ_CHECK_ARG(count > 0 && params_host && grads_host && sizes_host && offsets_host && slots_host, "az_adam_step: null table");
    AZ_CHECK_ARG(cfg->state_bits == 32 || cfg->state_bits == 8, "az_adam_step: moments in %d bits (32 or 8)", cfg->state_bits);
    AZ_CHECK_ARG(cfg->m_dev && cfg->v_dev && cfg->steps_dev && cfg->scratch_dev, "az_adam_step: null state");
    AZ_CHECK_ARG(cfg->state_bits == 32 || (cfg->m_scale_dev && cfg->v_scale_dev), "az_adam_step: 8-bit moments need scales");
    AZ_CHECK_ARG((uintptr_t)cfg->m_dev % 16 == 0 && (uintptr_t)cfg->v_dev % 16 == 0, "az_adam_step: the moments must be 16-byte aligned");
    AZ_CHECK_ARG(cfg->n_slots > 0 && cfg->n_slots <= 1 << 20, "az_adam_step: %d step counters (1 to 2^20)", cfg->n_slots);
    AZ_CHECK_ARG(!(cfg->max_norm > 0) || (cfg->n_partials >= 0 && (cfg->n_partials == 0 || cfg->partials_dev)), "az_adam_step: null partial sums");
    for (int32_t i = 0; i < count; ++i) {
        AZ_CHECK_ARG(slots_host[i] >= 0 && slots_host[i] < cfg->n_slots, "az_adam_step: step counter %d of %d", slots_host[i], cfg->n_slots);
        AZ_CHECK_ARG(sizes_host[i] >= 0 && offsets_host[i] >= 0 && offsets_host[i] % OPT_BLOCK == 0 && offsets_host[i] <= cfg->capacity &&
                         (sizes_host[i] + OPT_BLOCK - 1) / OPT_BLOCK * OPT_BLOCK <= cfg->capacity - offsets_host[i],
                     "az_adam_step: tensor %d does not fit the moments", i);
        AZ_CHECK_ARG(sizes_host[i] == 0 || (params_host[i] && params_host[i] % 4 == 0), "parameter %d is null or not aligned to 4 bytes", i);
    }
    float* scratch = (float*)cfg->scratch_dev;            // [0] clipping factor, then the tensors' factors
    OptHyper h;
    h.lr = cfg->lr;
    h.beta1 = cfg->beta1;
    h.beta2 = cfg->beta2;
    h.max_norm = cfg->max_norm;
    h.partials = cfg->partials_dev;
    h.n_partials = (uint32_t)cfg->n_partials;
    h.norm = cfg->norm_dev;
    h.coef = cfg->max_norm > 0 ? scratch : nullptr;
    h.steps = cfg->steps_dev;
    h.factors = (StepFactors*)(scratch + 4);
    h.seed_key = (uint32_t)cfg->seed * 0x9E3779B9u;
    AdamParams a;
    a.beta1 = (float)cfg->beta1;
    a.one_beta1 = (float)(1.0 - cfg->beta1);
    a.beta2 = (float)cfg->beta2;
    a.one_beta2 = (float)(1.0 - cfg->beta2);
    a.eps = (float)cfg->eps;
    a.decoupled = cfg->decoupled != 0;
    a.decay = a.decoupled ? (float)(1.0 - cfg->lr * cfg->weight_decay) : (float)cfg->weight_decay;
    a.coef = h.coef;
    a.factors = h.factors;
    a.m = cfg->m_dev;
    a.v = cfg->v_dev;
    a.m_scale = cfg->m_scale_dev;
    a.v_scale = cfg->v_scale_dev;
    for (int32_t at = 0; at < count; at += OPT_SLOTS) {
        SlotList l;
        const uint32_t k = (uint32_t)(count - at < OPT_SLOTS ? count - at : OPT_SLOTS);
        for (uint32_t i = 0; i < k; ++i) l.slot[i] = (uint32_t)slots_host[at + i];
        hipLaunchKernelGGL(k_adam_begin, dim3(1), dim3(1024), 0, (hipStream_t)stream, l, k, h);
        AZ_HIP(hipGetLastError());
    }
    return for_tables(count, params_host, grads_host, sizes_host, offsets_host, slots_host, [&](const OptTable& t, int64_t) -> int {
        if (cfg->state_bits == 32)
            hipLaunchKernelGGL(k_adam<32>, dim3(t.chunks), dim3(OPT_THREADS), 0, (hipStream_t)stream, t, a);
        else
            hipLaunchKernelGGL(k_adam<8>, dim3(t.chunks), dim3(OPT_THREADS), 0, (hipStream_t)stream, t, a);
        AZ_HIP(hipGetLastError());
        return AZ_OK;
    });
}
