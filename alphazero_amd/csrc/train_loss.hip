// Soft-target cross-entropy of a policy head and of an outcome head, with their gradients.
//
// Mathematics, per row with logits z, targets t, over the places that the mask keeps:
//   m = max z,  S = sum exp(z - m),  T = sum t,  U = sum t (m - z)
//   loss = T log S + U   (both terms positive: nothing cancels)      gradient = (T exp(z - m) / S - t) * upstream / rows
// One pass keeps (m, S, T, U) in registers: when the maximum grows by d, S shrinks by exp(-d) and U grows by d T.  A place
// whose target is zero adds nothing whatever its logit; a row that keeps nothing has loss 0 and gradient 0.
//
// Where the row fits a workgroup's registers (8192 actions) it is read once: first the maximum, then the sums, then the
// gradient for an upstream of 1, written by the same kernel.  The backward pass then only looks at the upstream and, if
// it is 1 (as it is when the loss itself is what backward() starts from), leaves what is there.  For another upstream, for
// longer rows and for a second backward pass the gradient is computed from the logits again, and in float16 always: there one
// that is divided by the rows and not yet multiplied with the program's loss scale would underflow.
//
// What bounds it: memory at large action spaces (k_loss_row at 8192 x 4001 in bfloat16 with a mask: 295 MB in 57 us,
// 5.2 TB/s), launches at small ones (1024 x 192: 4.0 + 2.8 + 2.6 us).  All sums in 32 bits; rows are added in 64 bits in a
// fixed order.
#include <math.h>

#include "train_common.h"

namespace az {

constexpr int LOSS_THREADS = 256;

struct LossParams {
    const void *policy, *wl;
    const float *target_pi, *target_wl;
    const uint8_t* mask;
    float *loss, *top, *inv, *total;   // [2n]: loss, m, 1 / S, T: the policy's rows, then the outcome's
    const float* upstream[3];  // gradients of (loss, policy loss, outcome loss), each may be null
    void *dpolicy, *dwl;
    int n, actions, outcomes;
};

struct RowSum {
    float m, S, T, U;
};

// exp(x) of an x that is not positive, to two last places; what would be below 2^-126 is 0.  2^y of y = x / ln 2 alone is off by
// |y| half-steps, so the rest of the product is kept and multiplied in.  (The library's expf: k_loss_row at 8192 x 4001 in
// bfloat16, the same inputs again, 53.6 us; this one 49.5.)
__device__ inline float exp_below(float x) {
    constexpr float INV_LN2 = (float)M_LOG2E, INV_LN2_REST = (float)(M_LOG2E - (double)INV_LN2);
    x = x < -150.f ? -150.f : x;               // (minus infinity has no rest; a NaN stays one)
    const float y = x * INV_LN2, rest = __builtin_fmaf(x, INV_LN2_REST, __builtin_fmaf(x, INV_LN2, -y));
    const float e = __builtin_amdgcn_exp2f(y);
    return __builtin_fmaf(e, rest * (float)M_LN2, e);
}

__device__ inline void absorb(RowSum& r, float z, float t) {          // z <= r.m
    if (z != -INFINITY) r.S += exp_below(z - r.m);
    r.T += t;
    if (t != 0.f) r.U += t * (z == -INFINITY ? INFINITY : r.m - z);
}

__device__ inline void raise(RowSum& r, float m) {
    if (m > r.m) {
        if (r.m != -INFINITY) {
            r.S *= exp_below(r.m - m);
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

// 1 / S; 0 where a row keeps nothing, or only logits of minus infinity, and has no target either.
__device__ inline float inverse(const RowSum& r) { return r.T == 0.f && r.S == 0.f ? 0.f : 1.f / r.S; }

__device__ inline void put_row(const LossParams& p, size_t at, const RowSum& r) {
    p.top[at] = r.m;
    p.inv[at] = inverse(r);
    p.total[at] = r.T;
    p.loss[at] = r.T == 0.f && r.U == 0.f && !(r.S != r.S) ? 0.f : r.T * logf(r.S) + r.U;
}

// weight: T / S; up: upstream / rows.  (Without targets the logits do not matter: z and m may both be minus infinity.)
__device__ inline float gradient(float z, float t, float m, float weight, float up) {
    return ((weight == 0.f ? 0.f : exp_below(z - m) * weight) - t) * up;
}

// One outcome row by one thread: two or three classes.
template <typename T, bool GRAD>
__device__ void outcome_forward(const LossParams& p, int row) {
    const T* z = (const T*)p.wl + (size_t)row * p.outcomes;
    const float* t = p.target_wl + (size_t)row * p.outcomes;
    RowSum r = {-INFINITY, 0.f, 0.f, 0.f};
    for (int i = 0; i < p.outcomes; ++i) {
        const float zi = (float)z[i];
        raise(r, zi);
        absorb(r, zi, t[i]);
    }
    put_row(p, (size_t)p.n + row, r);
    if (GRAD) {
        const float weight = inverse(r) * r.T, up = 1.f / (float)p.n;
        for (int i = 0; i < p.outcomes; ++i) ((T*)p.dwl)[(size_t)row * p.outcomes + i] = (T)gradient((float)z[i], t[i], r.m, weight, up);
    }
}

// Sums over a group's threads, in all of them.
template <int GROUP>
__device__ inline float group_max(float v, float* red) {
    v = lane_max<64>(v);
    if (GROUP == 64) return v;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < GROUP / 64; ++w) v = fmaxf(v, red[w]);
    return v;
}

// A row in the registers of GROUP threads, PIECES pieces of 16 bytes each (actions: at least one piece, at most
// GROUP * PIECES).  The last piece is moved back to end with the row: what it shares with its neighbour is left out of
// the sums and written twice, the same.
template <typename T, int GROUP, int PIECES, bool GRAD>
__global__ __launch_bounds__(LOSS_THREADS) void k_loss_row(const LossParams p, int policy_blocks) {
    constexpr int V = Pack<T>::V, ROWS = LOSS_THREADS / GROUP, WAVES = LOSS_THREADS / 64;
    __shared__ float red[4][WAVES];
    if ((int)blockIdx.x >= policy_blocks) {
        const int row = ((int)blockIdx.x - policy_blocks) * LOSS_THREADS + threadIdx.x;
        if (row < p.n) outcome_forward<T, GRAD>(p, row);
        return;
    }
    const int row = blockIdx.x * ROWS + threadIdx.x / GROUP, lane = threadIdx.x % GROUP;
    const size_t base = (size_t)(row < p.n ? row : 0) * p.actions;
    typedef uint8_t bytes_t __attribute__((ext_vector_type(V)));
    typedef bytes_t loose_bytes __attribute__((aligned(1)));
    typename Pack<T>::raw raw[PIECES];
    f32x4 t[PIECES][V / 4];
    bytes_t legal[PIECES];
    int off[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int at = (i * GROUP + lane) * V;
        off[i] = at < p.actions - V ? at : p.actions - V;
        raw[i] = *(const typename Pack<T>::loose*)((const T*)p.policy + base + off[i]);
#pragma unroll
        for (int k = 0; k < V / 4; ++k) t[i][k] = *(const f32x4_loose*)(p.target_pi + base + off[i] + 4 * k);
        if (p.mask) legal[i] = *(const loose_bytes*)(p.mask + base + off[i]);
    }
    float z[PIECES][V], top = -INFINITY;
    uint32_t keep[PIECES];                       // legal places of the piece
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        keep[i] = 0;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            z[i][k] = (float)raw[i][k];
            const bool on = !p.mask || legal[i][k];
            keep[i] |= (on ? 1u : 0u) << k;
            if (on) top = fmaxf(top, z[i][k]);
        }
    }
    top = group_max<GROUP>(top, red[3]);
    RowSum r = {top, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int own = (i * GROUP + lane) * V - off[i];            // the first place that is not the neighbour's
#pragma unroll
        for (int k = 0; k < V; ++k)
            if ((keep[i] >> k & 1) && k >= own) absorb(r, z[i][k], t[i][k / 4][k % 4]);
    }
    r.S = lane_sum<64>(r.S);
    r.T = lane_sum<64>(r.T);
    r.U = lane_sum<64>(r.U);
    if (GROUP > 64) {
        if ((threadIdx.x & 63) == 0) {
            red[0][threadIdx.x >> 6] = r.S;
            red[1][threadIdx.x >> 6] = r.T;
            red[2][threadIdx.x >> 6] = r.U;
        }
        __syncthreads();
        r.S = red[0][0];
        r.T = red[1][0];
        r.U = red[2][0];
        for (int w = 1; w < WAVES; ++w) {
            r.S += red[0][w];
            r.T += red[1][w];
            r.U += red[2][w];
        }
    }
    if (row >= p.n) return;
    if (lane == 0) put_row(p, row, r);
    if (GRAD) {
        const float weight = inverse(r) * r.T, up = 1.f / (float)p.n;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            if ((i * GROUP + lane) * V >= p.actions) break;
            typename Pack<T>::f32 g;
#pragma unroll
            for (int k = 0; k < V; ++k) g[k] = keep[i] >> k & 1 ? gradient(z[i][k], t[i][k / 4][k % 4], r.m, weight, up) : 0.f;
            *(typename Pack<T>::loose*)((T*)p.dpolicy + base + off[i]) = __builtin_convertvector(g, typename Pack<T>::raw);
        }
    }
}

// Any row: a wavefront up to 1024 actions, a workgroup above; (m, S, T, U) on the way.
template <typename T, int GROUP>
__global__ __launch_bounds__(LOSS_THREADS) void k_loss_forward(const LossParams p, int policy_blocks) {
    constexpr int V = Pack<T>::V, ROWS = LOSS_THREADS / GROUP;
    if ((int)blockIdx.x >= policy_blocks) {
        const int row = ((int)blockIdx.x - policy_blocks) * LOSS_THREADS + threadIdx.x;
        if (row < p.n) outcome_forward<T, false>(p, row);
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
        if (lane == 0 && row < p.n) put_row(p, row, r);
    } else {
        __shared__ RowSum part[LOSS_THREADS / 64];
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = r;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < LOSS_THREADS / 64; ++w) r = join(r, part[w]);
            put_row(p, row, r);
        }
    }
}

// Means over the rows: losses = (sum, policy, outcome).  Afterwards the first row's losses say that the gradients that were
// written are those for an upstream of 1.
__global__ __launch_bounds__(1024) void k_loss_sum(float* loss, int n, float* losses) {
    double a = 0.0, b = 0.0;
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += 1024) {
        a += loss[i];
        b += loss[(size_t)n + i];
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
        loss[0] = loss[n] = 1.f;
    }
}

__device__ inline float upstream_of(const LossParams& p, int which) {
    return (p.upstream[0] ? *p.upstream[0] : 0.f) + (p.upstream[which] ? *p.upstream[which] : 0.f);
}

// Which of V places the mask keeps, of the first `left`: its bytes in one load where all are there.
template <int V>
__device__ inline uint32_t legal_bits(const uint8_t* mask, int left) {
    typedef uint8_t bytes_t __attribute__((ext_vector_type(V)));
    typedef bytes_t loose_bytes __attribute__((aligned(1)));
    uint32_t bits = 0;
    if (mask && left >= V) {
        const bytes_t legal = *(const loose_bytes*)mask;
#pragma unroll
        for (int k = 0; k < V; ++k) bits |= (legal[k] ? 1u : 0u) << k;
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) bits |= (k < left && (!mask || mask[k]) ? 1u : 0u) << k;
    }
    return bits;
}

// The gradients from the logits.  ready: those for an upstream of 1 may be there already, from the forward kernel (the first
// row's loss, which nothing needs any more, says so for each head): they stay if the upstream is 1.  For another one they are
// computed anew, not multiplied: a gradient that is rounded already would be rounded twice, and a backward pass that is
// replayed without its forward pass would multiply what it has multiplied.  (8192 x 4001 in
// bfloat16 with a mask: 66 us, 4.4 TB/s; the multiplication took 20.)
template <typename T, int GROUP>
__global__ __launch_bounds__(LOSS_THREADS) void k_loss_backward(const LossParams p, int policy_blocks, int blocks, bool ready) {
    constexpr int V = Pack<T>::V, ROWS = LOSS_THREADS / GROUP;
    const float up_policy = upstream_of(p, 1), up_wl = upstream_of(p, 2);
    const bool leave_policy = ready && up_policy == 1.f && p.loss[0] == 1.f, leave_wl = ready && up_wl == 1.f && p.loss[p.n] == 1.f;
    if (leave_policy && leave_wl) return;
    if (blockIdx.x == 0 && threadIdx.x == 0) {       // (who reads this meanwhile has an upstream that is not 1)
        if (up_policy != 1.f) p.loss[0] = 0.f;
        if (up_wl != 1.f) p.loss[p.n] = 0.f;
    }
    const int lane = threadIdx.x % GROUP;
    for (int block = blockIdx.x; block < blocks; block += gridDim.x) {
        if (block >= policy_blocks) {
            const int row = (block - policy_blocks) * LOSS_THREADS + threadIdx.x;
            if (leave_wl || row >= p.n) continue;
            const float up = up_wl / (float)p.n, m = p.top[(size_t)p.n + row];
            const float weight = p.inv[(size_t)p.n + row] * p.total[(size_t)p.n + row];
            for (int i = 0; i < p.outcomes; ++i) {
                const size_t k = (size_t)row * p.outcomes + i;
                ((T*)p.dwl)[k] = (T)gradient((float)((const T*)p.wl)[k], p.target_wl[k], m, weight, up);
            }
            continue;
        }
        const int row = block * ROWS + threadIdx.x / GROUP;
        if (leave_policy || row >= p.n) continue;
        const float up = up_policy / (float)p.n, m = p.top[row], weight = p.inv[row] * p.total[row];
        const size_t at = (size_t)row * p.actions;
        for (int i = lane * V; i < p.actions; i += GROUP * V) {
            const int left = p.actions - i;
            auto z = load_pack((const T*)p.policy + at + i, left);
            const uint32_t legal = legal_bits<V>(p.mask ? p.mask + at + i : nullptr, left);
#pragma unroll
            for (int k = 0; k < V; k += 4) {
                const f32x4 q = load_pack(p.target_pi + at + i + k, left - k);
#pragma unroll
                for (int j = 0; j < 4; ++j) z[k + j] = legal >> (k + j) & 1 ? gradient(z[k + j], q[j], m, weight, up) : 0.f;
            }
            store_pack((T*)p.dpolicy + at + i, z, left);
        }
    }
}

// How many threads a row of so many actions gets, and how it is read: in registers, or (longer than 8192 actions, or
// shorter than a piece) in rounds.
template <typename T, bool GRAD>
static bool launch_row(const LossParams& p, hipStream_t s) {
    constexpr int V = Pack<T>::V;
    const dim3 block(LOSS_THREADS);
    const int outcome_blocks = (p.n + LOSS_THREADS - 1) / LOSS_THREADS, waves = (p.n + 3) / 4;
    if (p.actions < V || p.actions > 8192) return false;
    if (p.actions <= 512) hipLaunchKernelGGL((k_loss_row<T, 64, 512 / 64 / V, GRAD>), dim3(waves + outcome_blocks), block, 0, s, p, waves);
    else if (p.actions <= 2048) hipLaunchKernelGGL((k_loss_row<T, 256, 2048 / 256 / V, GRAD>), dim3(p.n + outcome_blocks), block, 0, s, p, p.n);
    else if (p.actions <= 4096) hipLaunchKernelGGL((k_loss_row<T, 256, 4096 / 256 / V, GRAD>), dim3(p.n + outcome_blocks), block, 0, s, p, p.n);
    else hipLaunchKernelGGL((k_loss_row<T, 256, 8192 / 256 / V, GRAD>), dim3(p.n + outcome_blocks), block, 0, s, p, p.n);
    return true;
}

template <typename T>
static int launch_loss(const LossParams& p, float* losses, bool backward, bool ready, hipStream_t s) {
    const int group = p.actions <= 1024 ? 64 : LOSS_THREADS;
    const int pb = (p.n + LOSS_THREADS / group - 1) / (LOSS_THREADS / group), ob = (p.n + LOSS_THREADS - 1) / LOSS_THREADS;
    const dim3 grid(pb + ob), block(LOSS_THREADS);
    if (backward) {
        // (most calls of a ready one find an upstream of 1 and leave: few workgroups, which take several blocks if they have to)
        const dim3 few(ready && pb + ob > 2048 ? 2048 : pb + ob);
        if (group == 64) hipLaunchKernelGGL((k_loss_backward<T, 64>), few, block, 0, s, p, pb, pb + ob, ready);
        else hipLaunchKernelGGL((k_loss_backward<T, LOSS_THREADS>), few, block, 0, s, p, pb, pb + ob, ready);
    } else {
        if (!(p.dpolicy ? launch_row<T, true>(p, s) : launch_row<T, false>(p, s))) {
            if (group == 64) hipLaunchKernelGGL((k_loss_forward<T, 64>), grid, block, 0, s, p, pb);
            else hipLaunchKernelGGL((k_loss_forward<T, LOSS_THREADS>), grid, block, 0, s, p, pb);
        }
        AZ_HIP(hipGetLastError());
        hipLaunchKernelGGL(k_loss_sum, dim3(1), dim3(1024), 0, s, p.loss, p.n, losses);
    }
    AZ_HIP(hipGetLastError());
    return AZ_OK;
}

// Whether the forward call can write the gradients.
static bool loss_ready(const az_loss_args* a) {
    return a->dtype != AZ_F16 && a->actions >= (a->dtype == AZ_F32 ? 4 : 8) && a->actions <= 8192;
}

static int loss_entry(const az_loss_args* a, bool backward, void* stream) {
    AZ_CHECK_ARG(a, "policy/value loss: null arguments");
    AZ_CHECK_ARG(a->n >= 1 && a->n <= 1 << 28, "policy/value loss: %lld rows (1 to 2^28)", (long long)a->n);
    AZ_CHECK_ARG(a->actions >= 1 && a->actions <= 1 << 28 && a->outcomes >= 1 && a->outcomes <= 4096,
                 "policy/value loss: %d actions, %d outcomes", a->actions, a->outcomes);
    AZ_CHECK_ARG((a->actions <= 512 ? (a->n + 3) / 4 : a->n) + a->n / LOSS_THREADS < MOST_BLOCKS,
                 "policy/value loss: %lld rows of %d actions are more than a launch takes", (long long)a->n, a->actions);
    AZ_CHECK_ARG(a->policy_dev && a->wl_dev && a->target_pi_dev && a->target_wl_dev && a->stats_dev && (uintptr_t)a->stats_dev % 16 == 0,
                 "policy/value loss: null input, or row statistics not aligned to 16 bytes");
    LossParams p;
    p.policy = a->policy_dev;
    p.wl = a->wl_dev;
    p.target_pi = a->target_pi_dev;
    p.target_wl = a->target_wl_dev;
    p.mask = a->mask_dev;
    p.loss = a->stats_dev;
    p.top = p.loss + 2 * a->n;
    p.inv = p.top + 2 * a->n;
    p.total = p.inv + 2 * a->n;
    for (int i = 0; i < 3; ++i) p.upstream[i] = a->upstream_dev[i];
    p.dpolicy = a->dpolicy_dev;
    p.dwl = a->dwl_dev;
    p.n = (int)a->n;
    p.actions = a->actions;
    p.outcomes = a->outcomes;
    if (backward) AZ_CHECK_ARG(p.dpolicy && p.dwl, "policy/value loss: null gradient");
    else AZ_CHECK_ARG(a->losses_dev, "policy/value loss: null output");
    AZ_CHECK_ARG(!p.dpolicy == !p.dwl, "policy/value loss: one gradient without the other");
    AZ_CHECK_ARG(backward ? !a->grads_ready || loss_ready(a) : !p.dpolicy || loss_ready(a),
                 "policy/value loss: the forward call writes no gradients of type %d with %d actions", a->dtype, a->actions);
    switch (a->dtype) {
        case AZ_F32: return launch_loss<float>(p, a->losses_dev, backward, a->grads_ready != 0, (hipStream_t)stream);
        case AZ_BF16: return launch_loss<__bf16>(p, a->losses_dev, backward, a->grads_ready != 0, (hipStream_t)stream);
        case AZ_F16: return launch_loss<_Float16>(p, a->losses_dev, backward, a->grads_ready != 0, (hipStream_t)stream);
    }
    AZ_FAIL(AZ_ERR_ARG, "policy/value loss: unknown type %d", a->dtype);
}

}  // namespace az

extern "C" int az_policy_value_loss_forward(const az_loss_args* args, void* stream) { return az::loss_entry(args, false, stream); }
extern "C" int az_policy_value_loss_backward(const az_loss_args* args, void* stream) { return az::loss_entry(args, true, stream); }
extern "C" int az_policy_value_loss_ready(const az_loss_args* args) { return args && az::loss_ready(args) ? 1 : 0; }
