// Soft-target cross-entropy of a policy head and of an outcome head, with their gradients.
//
// Mathematics, per row with logits z, targets t, over the places that the mask keeps:
//   m = max z,  S = sum exp(z - m),  T = sum t,  U = sum t (m - z)
//   loss = T log S + U   (both terms positive: nothing cancels)      gradient = (T exp(z - m) / S - t) * upstream / rows
// One pass keeps (m, S, T, U) in registers: when the maximum grows by d, S shrinks by exp(-d) and U grows by d T.  A place
// whose target is zero adds nothing whatever its logit; a row that keeps nothing has loss 0 and gradient 0.
//
// What bounds it: memory at large action spaces, launches at small ones.  All sums in 32 bits; rows are added in 64 bits
// in a fixed order.
#include <math.h>

#include "train_common.h"

namespace az {

constexpr int LOSS_THREADS = 256;

struct LossParams {
    const void *policy, *wl;
    const float *target_pi, *target_wl;
    const uint8_t* mask;
    float* stats;              // [2n][4]: m, 1 / S, T, loss: the policy's rows, then the outcome's
    const float* upstream[3];  // gradients of (loss, policy loss, outcome loss), each may be null
    void *dpolicy, *dwl;
    int n, actions, outcomes;
};

struct RowSum {
    float m, S, T, U;
};

__device__ inline void absorb(RowSum& r, float z, float t) {          // z <= r.m
    if (z != -INFINITY) r.S += __expf(z - r.m);
    r.T += t;
    if (t != 0.f) r.U += t * (z == -INFINITY ? INFINITY : r.m - z);
}

__device__ inline void raise(RowSum& r, float m) {
    if (m > r.m) {
        if (r.m != -INFINITY) {
            r.S *= __expf(r.m - m);
            r.U += (m - r.m) * r.T;
        }
        r.m = m;
    }
}

__device__ inline RowSum join(RowSum a, RowSum b) {
    const float m = fmaxf(a.m, b.m);
    raise(a, m);
    raise(b, m);
    return {m, a.S + b.S, a.T + b.T, a.U + b.U};
}

__device__ inline RowSum join_lanes(RowSum r) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1)
        r = join(r, {__shfl_xor(r.m, off), __shfl_xor(r.S, off), __shfl_xor(r.T, off), __shfl_xor(r.U, off)});
    return r;
}

__device__ inline f32x4 row_stats(const RowSum& r) {
    f32x4 s;
    s[0] = r.m;
    s[1] = r.T == 0.f && r.S == 0.f ? 0.f : 1.f / r.S;
    s[2] = r.T;
    s[3] = r.T == 0.f && r.U == 0.f && !(r.S != r.S) ? 0.f : r.T * logf(r.S) + r.U;
    return s;
}

// One outcome row by one thread: two or three classes.
template <typename T>
__device__ void outcome_forward(const LossParams& p, int row) {
    const T* z = (const T*)p.wl + (size_t)row * p.outcomes;
    const float* t = p.target_wl + (size_t)row * p.outcomes;
    RowSum r = {-INFINITY, 0.f, 0.f, 0.f};
    for (int i = 0; i < p.outcomes; ++i) {
        const float zi = (float)z[i];
        raise(r, zi);
        absorb(r, zi, t[i]);
    }
    *(f32x4*)(p.stats + 4 * ((size_t)p.n + row)) = row_stats(r);
}

// GROUP threads to a policy row: a wavefront up to 1024 actions, a workgroup above.
template <typename T, int GROUP>
__global__ __launch_bounds__(LOSS_THREADS) void k_loss_forward(const LossParams p, int policy_blocks) {
    constexpr int V = Pack<T>::V, ROWS = LOSS_THREADS / GROUP;
    if ((int)blockIdx.x >= policy_blocks) {
        const int row = ((int)blockIdx.x - policy_blocks) * LOSS_THREADS + threadIdx.x;
        if (row < p.n) outcome_forward<T>(p, row);
        return;
    }
    const int row = blockIdx.x * ROWS + threadIdx.x / GROUP, lane = threadIdx.x % GROUP;
    RowSum r = {-INFINITY, 0.f, 0.f, 0.f};
    if (row < p.n) {
        const size_t at = (size_t)row * p.actions;
        for (int i = lane * V; i < p.actions; i += GROUP * V) {
            const int left = p.actions - i;
            const auto z = load_pack((const T*)p.policy + at + i, left);
            float t[V];
            bool keep[V];
#pragma unroll
            for (int k = 0; k < V; k += 4) {
                const f32x4 q = load_pack(p.target_pi + at + i + k, left - k);
#pragma unroll
                for (int j = 0; j < 4; ++j) t[k + j] = q[j];
            }
#pragma unroll
            for (int k = 0; k < V; ++k) keep[k] = k < left && (!p.mask || p.mask[at + i + k]);
            float top = -INFINITY;
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (keep[k]) top = fmaxf(top, z[k]);
            raise(r, top);
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (keep[k]) absorb(r, z[k], t[k]);
        }
    }
    r = join_lanes(r);
    if (GROUP == 64) {
        if (lane == 0 && row < p.n) *(f32x4*)(p.stats + 4 * (size_t)row) = row_stats(r);
    } else {
        __shared__ RowSum part[LOSS_THREADS / 64];
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = r;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < LOSS_THREADS / 64; ++w) r = join(r, part[w]);
            *(f32x4*)(p.stats + 4 * (size_t)row) = row_stats(r);
        }
    }
}

// Means over the rows: losses = (sum, policy, outcome).
__global__ __launch_bounds__(1024) void k_loss_sum(const float* stats, int n, float* losses) {
    double a = 0.0, b = 0.0;
    for (int i = threadIdx.x; i < n; i += 1024) {
        a += stats[4 * (size_t)i + 3];
        b += stats[4 * ((size_t)n + i) + 3];
    }
    for (int off = 32; off; off >>= 1) {
        a += __shfl_xor(a, off);
        b += __shfl_xor(b, off);
    }
    __shared__ double part[2][16];
    if ((threadIdx.x & 63) == 0) {
        part[0][threadIdx.x >> 6] = a;
        part[1][threadIdx.x >> 6] = b;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) {
            a += part[0][w];
            b += part[1][w];
        }
        losses[0] = (float)((a + b) / n);
        losses[1] = (float)(a / n);
        losses[2] = (float)(b / n);
    }
}

__device__ inline float upstream_of(const LossParams& p, int which) {
    return ((p.upstream[0] ? *p.upstream[0] : 0.f) + (p.upstream[which] ? *p.upstream[which] : 0.f)) / (float)p.n;
}

template <typename T, int GROUP>
__global__ __launch_bounds__(LOSS_THREADS) void k_loss_backward(const LossParams p, int policy_blocks) {
    constexpr int V = Pack<T>::V, ROWS = LOSS_THREADS / GROUP;
    if ((int)blockIdx.x >= policy_blocks) {
        const int row = ((int)blockIdx.x - policy_blocks) * LOSS_THREADS + threadIdx.x;
        if (row >= p.n) return;
        const float up = upstream_of(p, 2);
        const f32x4 s = *(const f32x4*)(p.stats + 4 * ((size_t)p.n + row));
        for (int i = 0; i < p.outcomes; ++i) {
            const size_t k = (size_t)row * p.outcomes + i;
            ((T*)p.dwl)[k] = (T)((__expf((float)((const T*)p.wl)[k] - s[0]) * s[1] * s[2] - p.target_wl[k]) * up);
        }
        return;
    }
    const int row = blockIdx.x * ROWS + threadIdx.x / GROUP, lane = threadIdx.x % GROUP;
    if (row >= p.n) return;
    const float up = upstream_of(p, 1);
    const f32x4 s = *(const f32x4*)(p.stats + 4 * (size_t)row);
    const float weight = s[1] * s[2];
    const size_t at = (size_t)row * p.actions;
    for (int i = lane * V; i < p.actions; i += GROUP * V) {
        const int left = p.actions - i;
        auto z = load_pack((const T*)p.policy + at + i, left);
#pragma unroll
        for (int k = 0; k < V; k += 4) {
            const f32x4 q = load_pack(p.target_pi + at + i + k, left - k);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool keep = k + j < left && (!p.mask || p.mask[at + i + k + j]);
                z[k + j] = keep ? (__expf(z[k + j] - s[0]) * weight - q[j]) * up : 0.f;
            }
        }
        store_pack((T*)p.dpolicy + at + i, z, left);
    }
}

template <typename T>
static int launch_loss(const LossParams& p, float* losses, bool backward, hipStream_t s) {
    const int group = p.actions <= 1024 ? 64 : LOSS_THREADS;
    const int pb = (p.n + LOSS_THREADS / group - 1) / (LOSS_THREADS / group), ob = (p.n + LOSS_THREADS - 1) / LOSS_THREADS;
    const dim3 grid(pb + ob), block(LOSS_THREADS);
    if (backward) {
        if (group == 64) hipLaunchKernelGGL((k_loss_backward<T, 64>), grid, block, 0, s, p, pb);
        else hipLaunchKernelGGL((k_loss_backward<T, LOSS_THREADS>), grid, block, 0, s, p, pb);
    } else {
        if (group == 64) hipLaunchKernelGGL((k_loss_forward<T, 64>), grid, block, 0, s, p, pb);
        else hipLaunchKernelGGL((k_loss_forward<T, LOSS_THREADS>), grid, block, 0, s, p, pb);
        AZ_HIP(hipGetLastError());
        hipLaunchKernelGGL(k_loss_sum, dim3(1), dim3(1024), 0, s, p.stats, p.n, losses);
    }
    AZ_HIP(hipGetLastError());
    return AZ_OK;
}

static int loss_entry(const az_loss_args* a, bool backward, void* stream) {
    AZ_CHECK_ARG(a, "policy/value loss: null arguments");
    AZ_CHECK_ARG(a->n >= 1 && a->n <= 1 << 28, "policy/value loss: %lld rows (1 to 2^28)", (long long)a->n);
    AZ_CHECK_ARG(a->actions >= 1 && a->actions <= 1 << 28 && a->outcomes >= 1 && a->outcomes <= 4096,
                 "policy/value loss: %d actions, %d outcomes", a->actions, a->outcomes);
    AZ_CHECK_ARG(a->policy_dev && a->wl_dev && a->target_pi_dev && a->target_wl_dev && a->stats_dev && (uintptr_t)a->stats_dev % 16 == 0,
                 "policy/value loss: null input, or row statistics not aligned to 16 bytes");
    LossParams p;
    p.policy = a->policy_dev;
    p.wl = a->wl_dev;
    p.target_pi = a->target_pi_dev;
    p.target_wl = a->target_wl_dev;
    p.mask = a->mask_dev;
    p.stats = a->stats_dev;
    for (int i = 0; i < 3; ++i) p.upstream[i] = a->upstream_dev[i];
    p.dpolicy = a->dpolicy_dev;
    p.dwl = a->dwl_dev;
    p.n = (int)a->n;
    p.actions = a->actions;
    p.outcomes = a->outcomes;
    if (backward) AZ_CHECK_ARG(p.dpolicy && p.dwl, "policy/value loss: null gradient");
    else AZ_CHECK_ARG(a->losses_dev, "policy/value loss: null output");
    switch (a->dtype) {
        case AZ_F32: return launch_loss<float>(p, a->losses_dev, backward, (hipStream_t)stream);
        case AZ_BF16: return launch_loss<__bf16>(p, a->losses_dev, backward, (hipStream_t)stream);
        case AZ_F16: return launch_loss<_Float16>(p, a->losses_dev, backward, (hipStream_t)stream);
    }
    AZ_FAIL(AZ_ERR_ARG, "policy/value loss: unknown type %d", a->dtype);
}

}  // namespace az

extern "C" int az_policy_value_loss_forward(const az_loss_args* args, void* stream) { return az::loss_entry(args, false, stream); }
extern "C" int az_policy_value_loss_backward(const az_loss_args* args, void* stream) { return az::loss_entry(args, true, stream); }
