// Adam / AdamW over many tensors in a few launches, moments in 32 bits or in 8, gradient clipping by the global norm.
//
// Mathematics, per element (t: the tensor's step counter after this step):
//   c = min(1, max_norm / (|g| + 1e-6))                  |g| over all gradients, summed in 64 bits
//   g = c g (+ wd p: weight decay in the gradient)        m = b1 m + (1 - b1) g        v = b2 v + (1 - b2) g^2
//   p = p (- lr wd p: decoupled decay) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// Every operation on the moments is rounded on its own to 32 bits (this file is built without contraction, the root is
// correctly rounded, denormals too), so they are the same numbers as the same operations in elementary tensor code, and so are
// the codes that they become in 8 bits.  The quotient is a product with the hardware's reciprocal: one last place of the update.
//
// What bounds it: memory.  A 32-bit step reads 16 and writes 12 bytes per weight, an 8-bit one 10 and 6; clipping reads
// the gradients once more.  Measured: k_adam on the 20x128 network's 8.0 M weights 41 us in 32 bits (5.5 TB/s), 30 us in
// 8 (4.3 TB/s; the codes' 80 instructions a weight are 20 us of it); on the 28 M of 20x256 in 8 bits 88 us (5.1 TB/s);
// k_adam_begin 9 us with the norm of 8.0 M gradients, 5 us without.
// Layout: a workgroup takes a piece of OPT_CHUNK elements of one tensor.  Which one is in a table that is made once, in
// device memory; the tensors' addresses travel in the kernel arguments (OPT_TABLE tensors a launch, so that the default
// network's 214 are one), nothing is uploaded per step: it can be captured, and tensors may move between steps.
// Two launches make a step: k_adam_begin (step counters and what follows from them, partial sums of squares) and k_adam,
// whose workgroups each add the partial sums themselves, in the same order, while their own loads are under way.
#include <math.h>

#include <type_traits>

#include "train_common.h"

namespace az {

constexpr int OPT_THREADS = 256;
constexpr int OPT_CHUNK = AZ_OPTIM_CHUNK;          // elements of one tensor that one workgroup takes
constexpr int OPT_BLOCK = AZ_OPTIM_PAD;            // elements that share a scale: one wavefront x 4
constexpr int OPT_ROUNDS = OPT_CHUNK / (OPT_THREADS * 4);
constexpr int OPT_TABLE = 240;                     // 16 bytes each: 3.75 of the 4 KB of kernel arguments
constexpr int OPT_GROUPS = AZ_OPTIM_GROUPS;
constexpr int OPT_SUMS = 1024;                     // partial sums per OPT_TABLE tensors, at most (256: k_adam_begin 13 us at 20x128, 512: 9.6, 1024: 9.1)
static_assert(OPT_CHUNK % (OPT_THREADS * 4) == 0 && OPT_BLOCK == 256, "a wavefront covers one block of a moment");

struct GradTable {
    uint64_t grad[OPT_TABLE];       // 0: none, the tensor is left alone
};

struct TensorTable {
    uint64_t grad[OPT_TABLE], param[OPT_TABLE];
};

struct StepFactors {                // per tensor, from its step counter
    float step_size, inv_root_bias2;
    uint32_t key;
};

struct GroupRates {
    double lr, beta1, beta2;
    uint32_t end;                   // first tensor after the group
};

struct BeginParams {
    GroupRates group[OPT_GROUPS];
    const az_adam_piece* pieces;
    uint32_t first_tensor, tensors, n_pieces, seed_key;
    double* partials;
    float* steps;
    StepFactors* factors;
};

struct AdamParams {
    float beta1, one_beta1, beta2, one_beta2, eps, decay;   // decay: wd, or 1 - lr wd
    int decoupled;
    const az_adam_piece* pieces;
    uint32_t first_tensor;
    const StepFactors* factors;
    double max_norm;                // 0: no clipping
    const double* partials;
    uint32_t n_partials;
    float* norm;                    // |g| out (may be null)
    void *m, *v;
    float *m_scale, *v_scale;
};

// f(whether the piece is whole): a whole piece's loads are issued together, the last one of a tensor goes round by round.
template <typename F>
__device__ inline void with_whole(const az_adam_piece& c, F&& f) {
    if (c.n == OPT_CHUNK) f(std::true_type());
    else f(std::false_type());
}

template <bool WHOLE>
__device__ inline f32x4 load_four(const float* p, int i, const az_adam_piece& c) {
    return WHOLE ? *(const f32x4_loose*)(p + i) : load_pack(p + i, (int)c.n - i);
}

// The sum of a workgroup's v in all its threads, always in the same order.
__device__ inline double block_sum(double v) {
    __shared__ double part[OPT_THREADS / 64];
    for (int off = 32; off; off >>= 1) v += __shfl_xor(v, off);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
    for (int w = 1; w < OPT_THREADS / 64; ++w) v += part[w];
    return v;
}

// The last workgroup: the tensors' step counters and what follows from them.  The others: partial sums of squares, in
// 64 bits (the products are exact there): the norm of 8 M gradients whose sizes lie decades apart, and a clipping factor
// that does not depend on the order of the sum.
__global__ __launch_bounds__(OPT_THREADS) void k_adam_begin(const GradTable t, const BeginParams h) {
    if (blockIdx.x == gridDim.x - 1) {
        for (uint32_t i = threadIdx.x; i < h.tensors; i += OPT_THREADS) {
            if (!t.grad[i]) continue;
            const uint32_t tensor = h.first_tensor + i;
            int g = 0;
            while (h.group[g].end <= tensor) ++g;
            const float step = h.steps[tensor] + 1.f;
            h.steps[tensor] = step;
            StepFactors f;
            f.step_size = (float)(h.group[g].lr / (1.0 - pow(h.group[g].beta1, (double)step)));
            f.inv_root_bias2 = 1.f / (float)sqrt(1.0 - pow(h.group[g].beta2, (double)step));
            f.key = h.seed_key + (uint32_t)step * 0x85EBCA6Bu;
            h.factors[tensor] = f;
        }
        return;
    }
    double s = 0.0;
    for (uint32_t piece = blockIdx.x; piece < h.n_pieces; piece += gridDim.x - 1) {
        const az_adam_piece c = h.pieces[piece];
        const float* g = (const float*)t.grad[c.tensor - h.first_tensor];
        if (!g) continue;
        g += (size_t)c.chunk * OPT_CHUNK;
        with_whole(c, [&](auto whole) {
            f32x4 v[OPT_ROUNDS];
#pragma unroll
            for (int it = 0; it < OPT_ROUNDS; ++it) v[it] = load_four<decltype(whole)::value>(g, (it * OPT_THREADS + threadIdx.x) * 4, c);
#pragma unroll
            for (int it = 0; it < OPT_ROUNDS; ++it)
#pragma unroll
                for (int k = 0; k < 4; ++k) s += (double)v[it][k] * (double)v[it][k];
        });
    }
    s = block_sum(s);
    if (threadIdx.x == 0) h.partials[blockIdx.x] = s;
}

// The clipping factor, from all partial sums.
__device__ inline float clip_factor(const AdamParams& a) {
    constexpr int EACH = OPT_SUMS / OPT_THREADS;       // of one launch's sums, loaded together
    double s = 0.0;
    for (uint32_t i = threadIdx.x; i < a.n_partials; i += OPT_SUMS) {
        double part[EACH];
#pragma unroll
        for (int u = 0; u < EACH; ++u) part[u] = a.partials[i + u * OPT_THREADS < a.n_partials ? i + u * OPT_THREADS : i];
#pragma unroll
        for (int u = 0; u < EACH; ++u) s += i + u * OPT_THREADS < a.n_partials ? part[u] : 0.0;
    }
    const double norm = sqrt(block_sum(s)), c = a.max_norm / (norm + 1e-6);
    if (a.norm && blockIdx.x == 0 && threadIdx.x == 0) *a.norm = (float)norm;
    return (float)(c > 1.0 ? 1.0 : c);             // a NaN stays one
}

// ---- moments in 8 bits -------------------------------------------------------------------------------------------
// 256 values share a power of two that puts their largest in (224, 448]; each is an e4m3 code times it: 3 bits of
// mantissa over 17 binades, both directions of the scaling exact.  m is held as itself, v as its root: the root is what
// the update divides by, and squaring 17 binades would lose the small ones.  A decaying average moves by less than half
// a code's step (6 %) per step, so rounding to nearest would freeze it: values are rounded at random, up with the
// probability of the way they have gone.  That keeps the averages of m and of the root right, not those of the root's square:
// with beta2 = 0.999 v settles 3 to 5 % above its average for weights whose gradients are up to four decades smaller than the
// largest of their 256 (their mean update is off by 1 %), 50 to 80 % above it at five.  A root that is not zero never becomes
// zero (the update would divide by eps alone): more than 5.4 decades below the largest it is the smallest code, far too
// large, and such weights hardly move (13 % of the update at six decades, 1 % at seven).  What is not finite becomes the code of
// NaN.

// The largest finite magnitude of the wavefront's 256 values, as the bits of a float (those order like integers).
__device__ inline uint32_t wave_max(uint32_t v) {
#define AZ_MAX_DPP(CTRL) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true))
    AZ_MAX_DPP(0xB1);
    AZ_MAX_DPP(0x4E);
    AZ_MAX_DPP(0x141);
    AZ_MAX_DPP(0x140);
#undef AZ_MAX_DPP
    v = max(v, (uint32_t)__shfl_xor((int)v, 16));
    return max(v, (uint32_t)__shfl_xor((int)v, 32));
}

__device__ inline uint32_t block_top(const f32x4 x) {
    constexpr uint32_t INF = 0x7F800000u;
    uint32_t b[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) b[k] = __float_as_uint(x[k]) & 0x7FFFFFFFu;
    const uint32_t top = wave_max(max(max(b[0], b[1]), max(b[2], b[3])));
    if (top < INF) return top;               // the same in every lane
#pragma unroll
    for (int k = 0; k < 4; ++k) b[k] = b[k] < INF ? b[k] : 0;
    return wave_max(max(max(b[0], b[1]), max(b[2], b[3])));
}

__device__ inline int scale_exponent(uint32_t top) {
    const int k = (int)(top >> 23) - 127 - 8 + ((top & 0x7FFFFFu) > 0x600000u);
    return k < -108 ? -108 : k;
}

__device__ inline float pow2(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }

// The magnitude of x in units of the scale as a code, rounded by 16 random bits.  From 2^-6 on a code is the float's exponent
// and its first three mantissa bits: the random bits go on top of what is cut off, as an integer.  Below, codes are
// multiples of 2^-9.  What is not finite ends above the largest code.
__device__ inline uint32_t encode(float x, float inv_scale, uint32_t r16) {
    const float y = fabsf(x) * inv_scale;
    const uint32_t code = ((__float_as_uint(y) + (r16 << 4)) >> 20) - (120u << 3);
    const uint32_t small = (uint32_t)__builtin_fmaf((float)r16, 1.f / 65536.f, y * 512.f);     // both products exact
    return y < 0.015625f ? small : min(code, 0x7Fu);
}

__device__ inline f32x4 decode(uint32_t codes, float scale) {
    f32x4 r;
    r[0] = __builtin_amdgcn_cvt_f32_fp8(codes, 0) * scale;
    r[1] = __builtin_amdgcn_cvt_f32_fp8(codes, 1) * scale;
    r[2] = __builtin_amdgcn_cvt_f32_fp8(codes, 2) * scale;
    r[3] = __builtin_amdgcn_cvt_f32_fp8(codes, 3) * scale;
    return r;
}

// (A published mix of 32 bits with little bias, C. Wellons 2018: two rounds of xor-shift and multiply.)
__device__ inline uint32_t mix32(uint32_t z) {
    z = (z ^ (z >> 16)) * 0x7FEB352Du;
    z = (z ^ (z >> 15)) * 0x846CA68Bu;
    return z ^ (z >> 16);
}

template <int BITS>
__global__ __launch_bounds__(OPT_THREADS) void k_adam(const TensorTable t, const AdamParams a) {
    const az_adam_piece c = a.pieces[blockIdx.x];
    const bool clip = a.max_norm > 0.0;
    const float* gp = (const float*)t.grad[c.tensor - a.first_tensor];
    if (!gp) {
        if (clip && blockIdx.x == 0) clip_factor(a);                // the norm is this workgroup's to write
        return;
    }
    gp += (size_t)c.chunk * OPT_CHUNK;
    float* pp = (float*)t.param[c.tensor - a.first_tensor] + (size_t)c.chunk * OPT_CHUNK;
    const size_t at = (size_t)c.offset * OPT_BLOCK;                 // the piece's place in the moments
    const StepFactors f = a.factors[c.tensor];
    float coef = 1.f;
    with_whole(c, [&](auto whole) {
        constexpr bool WHOLE = decltype(whole)::value;
        constexpr int AHEAD = WHOLE ? OPT_ROUNDS : 1;          // rounds whose loads are under way together
        if (!WHOLE && clip) coef = clip_factor(a);
#pragma unroll
        for (int it0 = 0; it0 < OPT_ROUNDS; it0 += AHEAD) {
            f32x4 p[AHEAD], g[AHEAD], m[AHEAD], v[AHEAD];
            uint32_t cm[AHEAD], cv[AHEAD];
            float sm[AHEAD], sv[AHEAD];
            // a wavefront whose block is past the end of the tensor is done (the moments run on to a whole block)
            if (!WHOLE && (int)c.n <= (it0 * OPT_THREADS + (int)(threadIdx.x & ~63u)) * 4) return;
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int i = ((it0 + u) * OPT_THREADS + threadIdx.x) * 4;
                p[u] = load_four<WHOLE>(pp, i, c);
                g[u] = load_four<WHOLE>(gp, i, c);
                if (BITS == 32) {
                    m[u] = *(const f32x4*)((const float*)a.m + at + i);
                    v[u] = *(const f32x4*)((const float*)a.v + at + i);
                } else {
                    cm[u] = *(const uint32_t*)((const uint8_t*)a.m + at + i);
                    cv[u] = *(const uint32_t*)((const uint8_t*)a.v + at + i);
                    sm[u] = a.m_scale[(at + i) / OPT_BLOCK];
                    sv[u] = a.v_scale[(at + i) / OPT_BLOCK];
                }
            }
            if (WHOLE && clip) coef = clip_factor(a);
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int i = ((it0 + u) * OPT_THREADS + threadIdx.x) * 4;
                if (BITS == 8) {
                    m[u] = decode(cm[u], sm[u]);
                    v[u] = decode(cv[u], sv[u]);
                }
                f32x4 root;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float gk = g[u][k], pk = p[u][k];
                    if (clip) gk = gk * coef;
                    if (a.decoupled) pk = pk * a.decay;
                    else if (a.decay != 0.f) gk = gk + pk * a.decay;
                    const float vk = BITS == 32 ? v[u][k] : v[u][k] * v[u][k];
                    m[u][k] = m[u][k] * a.beta1 + gk * a.one_beta1;
                    v[u][k] = vk * a.beta2 + gk * gk * a.one_beta2;
                    root[k] = sqrtf(v[u][k]);
                    p[u][k] = pk - m[u][k] * __builtin_amdgcn_rcpf(root[k] * f.inv_root_bias2 + a.eps) * f.step_size;
                }
                if (WHOLE) *(f32x4_loose*)(pp + i) = p[u];
                else store_pack(pp + i, p[u], (int)c.n - i);
                if (BITS == 32) {
                    *(f32x4*)((float*)a.m + at + i) = m[u];
                    *(f32x4*)((float*)a.v + at + i) = v[u];
                } else {
                    const int km = scale_exponent(block_top(m[u])), kv = scale_exponent(block_top(root));
                    uint32_t em = 0, ev = 0;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t place = (uint32_t)(at + i + k), r = mix32(place + f.key);
                        em |= (encode(m[u][k], pow2(-km), r & 0xFFFF) | __float_as_uint(m[u][k]) >> 31 << 7) << (8 * k);
                        const uint32_t code = encode(root[k], pow2(-kv), r >> 16);
                        ev |= max(code, min(__float_as_uint(root[k]), 1u)) << (8 * k);        // at least 1 unless the root is 0
                    }
                    *(uint32_t*)((uint8_t*)a.m + at + i) = em;
                    *(uint32_t*)((uint8_t*)a.v + at + i) = ev;
                    if ((threadIdx.x & 63) == 0) {
                        a.m_scale[(at + i) / OPT_BLOCK] = pow2(km);
                        a.v_scale[(at + i) / OPT_BLOCK] = pow2(kv);
                    }
                }
            }
        }
    });
}

static int64_t pieces_of(int64_t n) { return (n + OPT_CHUNK - 1) / OPT_CHUNK; }

// Calls launch(first tensor, tensors, first piece, pieces) for ranges of OPT_TABLE tensors of [begin, end).
template <typename F>
static int for_ranges(int32_t begin, int32_t end, const int64_t* sizes, F&& launch) {
    int64_t piece = 0;
    for (int32_t i = 0; i < begin; ++i) piece += pieces_of(sizes[i]);
    for (int32_t i = begin; i < end; i += OPT_TABLE) {
        const int32_t k = end - i < OPT_TABLE ? end - i : OPT_TABLE;
        int64_t n = 0;
        for (int32_t j = i; j < i + k; ++j) n += pieces_of(sizes[j]);
        if (n) {
            const int rc = launch(i, k, piece, (uint32_t)n);
            if (rc != AZ_OK) return rc;
        }
        piece += n;
    }
    return AZ_OK;
}

}  // namespace az

using namespace az;

extern "C" int64_t az_adam_plan(int32_t count, const int64_t* sizes_host, int64_t* offsets_host, az_adam_piece* pieces_host) {
    AZ_CHECK_ARG(count >= 0 && (count == 0 || sizes_host), "az_adam_plan: null sizes");
    int64_t at = 0, piece = 0;
    for (int32_t i = 0; i < count; ++i) {
        AZ_CHECK_ARG(sizes_host[i] >= 0 && sizes_host[i] <= int64_t(1) << 38, "az_adam_plan: tensor %d has %lld elements", i, (long long)sizes_host[i]);
        if (offsets_host) offsets_host[i] = at;
        for (int64_t k = 0; k < pieces_of(sizes_host[i]); ++k, ++piece) {
            if (!pieces_host) continue;
            const int64_t left = sizes_host[i] - k * OPT_CHUNK;
            pieces_host[piece] = {(uint32_t)i, (uint32_t)k, (uint32_t)((at + k * OPT_CHUNK) / OPT_BLOCK), (uint32_t)(left < OPT_CHUNK ? left : OPT_CHUNK)};
        }
        at += (sizes_host[i] + OPT_BLOCK - 1) / OPT_BLOCK * OPT_BLOCK;
    }
    AZ_CHECK_ARG(at / OPT_BLOCK <= 0xFFFFFFFF && piece <= MOST_BLOCKS, "az_adam_plan: too many elements");
    if (offsets_host) offsets_host[count] = at;
    return piece;
}

extern "C" int64_t az_adam_scratch(int32_t count) {
    AZ_CHECK_ARG(count >= 0, "az_adam_scratch: %d tensors", count);
    return (int64_t)((count + OPT_TABLE - 1) / OPT_TABLE) * OPT_SUMS * sizeof(double) + (int64_t)count * sizeof(StepFactors);
}

extern "C" int az_adam_step(const az_adam_config* cfg, int32_t n_groups, const az_adam_group* groups, int32_t count, const uint64_t* params_host,
                            const uint64_t* grads_host, const int64_t* sizes_host, void* stream) {
    AZ_CHECK_ARG(cfg && groups && n_groups >= 1 && n_groups <= OPT_GROUPS, "az_adam_step: null config, or %d groups (1 to %d)", n_groups, OPT_GROUPS);
    AZ_CHECK_ARG(count >= 0 && (count == 0 || (sizes_host && grads_host && params_host)), "az_adam_step: null table");
    int64_t pieces = 0;
    for (int32_t i = 0; i < count; ++i) {
        AZ_CHECK_ARG(sizes_host[i] >= 0 && sizes_host[i] <= int64_t(1) << 38, "az_adam_step: tensor %d has %lld elements", i, (long long)sizes_host[i]);
        pieces += pieces_of(sizes_host[i]);
        if (!grads_host[i] || !sizes_host[i]) continue;
        AZ_CHECK_ARG(grads_host[i] % 4 == 0, "az_adam_step: gradient %d is not aligned to 4 bytes", i);
        AZ_CHECK_ARG(params_host[i] && params_host[i] % 4 == 0, "az_adam_step: parameter %d is null or not aligned to 4 bytes", i);
    }
    for (int32_t g = 0, at = 0; g < n_groups; at = groups[g++].end)
        AZ_CHECK_ARG(groups[g].end >= at && (g + 1 < n_groups ? groups[g].end <= count : groups[g].end == count),
                     "az_adam_step: group %d ends at %d of %d tensors", g, groups[g].end, count);
    if (pieces == 0) return AZ_OK;
    AZ_CHECK_ARG(pieces <= MOST_BLOCKS, "az_adam_step: too many elements");
    AZ_CHECK_ARG(cfg->state_bits == 32 || cfg->state_bits == 8, "az_adam_step: moments in %d bits (32 or 8)", cfg->state_bits);
    AZ_CHECK_ARG(cfg->m_dev && cfg->v_dev && cfg->steps_dev && cfg->scratch_dev && cfg->pieces_dev, "az_adam_step: null state");
    AZ_CHECK_ARG(cfg->state_bits == 32 || (cfg->m_scale_dev && cfg->v_scale_dev), "az_adam_step: 8-bit moments need scales");
    AZ_CHECK_ARG((uintptr_t)cfg->m_dev % 16 == 0 && (uintptr_t)cfg->v_dev % 16 == 0 && (uintptr_t)cfg->scratch_dev % 16 == 0,
                 "az_adam_step: moments and scratch memory must be 16-byte aligned");
    const bool clip = cfg->max_norm > 0;
    double* partials = (double*)cfg->scratch_dev;         // then the tensors' factors
    StepFactors* factors = (StepFactors*)(partials + (size_t)((count + OPT_TABLE - 1) / OPT_TABLE) * OPT_SUMS);
    uint32_t n_partials = 0;
    int rc = for_ranges(0, count, sizes_host, [&](int32_t first, int32_t k, int64_t piece, uint32_t n) -> int {
        GradTable t;
        for (int32_t i = 0; i < k; ++i) t.grad[i] = sizes_host[first + i] ? grads_host[first + i] : 0;
        BeginParams b;
        for (int32_t g = 0; g < n_groups; ++g) b.group[g] = {groups[g].lr, groups[g].beta1, groups[g].beta2, (uint32_t)groups[g].end};
        b.pieces = cfg->pieces_dev + piece;
        b.first_tensor = (uint32_t)first;
        b.tensors = (uint32_t)k;
        b.n_pieces = n;
        b.seed_key = (uint32_t)cfg->seed * 0x9E3779B9u;
        b.partials = partials + n_partials;
        b.steps = cfg->steps_dev;
        b.factors = factors;
        const uint32_t sums = !clip ? 0 : n < (uint32_t)OPT_SUMS ? n : OPT_SUMS;
        hipLaunchKernelGGL(k_adam_begin, dim3(sums + 1), dim3(OPT_THREADS), 0, (hipStream_t)stream, t, b);
        AZ_HIP(hipGetLastError());
        n_partials += sums;
        return AZ_OK;
    });
    float* norm = cfg->norm_dev;
    for (int32_t g = 0, begin = 0; g < n_groups && rc == AZ_OK; begin = groups[g++].end) {
        AdamParams a;
        a.beta1 = (float)groups[g].beta1;
        a.one_beta1 = (float)(1.0 - groups[g].beta1);
        a.beta2 = (float)groups[g].beta2;
        a.one_beta2 = (float)(1.0 - groups[g].beta2);
        a.eps = (float)groups[g].eps;
        a.decoupled = groups[g].decoupled != 0;
        a.decay = a.decoupled ? (float)(1.0 - groups[g].lr * groups[g].weight_decay) : (float)groups[g].weight_decay;
        a.factors = factors;
        a.max_norm = clip ? cfg->max_norm : 0.0;
        a.partials = partials;
        a.n_partials = n_partials;
        a.m = cfg->m_dev;
        a.v = cfg->v_dev;
        a.m_scale = cfg->m_scale_dev;
        a.v_scale = cfg->v_scale_dev;
        rc = for_ranges(begin, groups[g].end, sizes_host, [&](int32_t first, int32_t k, int64_t piece, uint32_t n) -> int {
            TensorTable t;
            for (int32_t i = 0; i < k; ++i) {
                t.grad[i] = grads_host[first + i];
                t.param[i] = params_host[first + i];
            }
            a.pieces = cfg->pieces_dev + piece;
            a.first_tensor = (uint32_t)first;
            a.norm = norm;
            norm = nullptr;                               // written once
            if (cfg->state_bits == 32)
                hipLaunchKernelGGL(k_adam<32>, dim3(n), dim3(OPT_THREADS), 0, (hipStream_t)stream, t, a);
            else
                hipLaunchKernelGGL(k_adam<8>, dim3(n), dim3(OPT_THREADS), 0, (hipStream_t)stream, t, a);
            AZ_HIP(hipGetLastError());
            return AZ_OK;
        });
    }
    return rc;
}
