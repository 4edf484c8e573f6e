// Batch normalisation with ReLU, and the end of a squeeze-excitation residual block, forward and backward.
//
// Mathematics, for a convolution's output x (n boards, c channels, hw places), mu and 1/s from the batch (or the running
// statistics), xc = x - mu:
//   y = weight xc / s + bias                                          plain:  out = relu(y)
//   q = mean_hw y,  h = relu(fc1 q + b1),  (w, b) = fc2 h + b2        gated:  out = relu(y sigmoid(w) + b + residual)
// Forward: one pass over x takes the mean and the centred sum of squares of every board and channel ("row"); from these
// come the batch's statistics and the squeeze q, so x is read once more only, for out = relu(A x + B (+ residual)) with
// A, B per row (gated) or per channel (plain).
// Backward, with gm = grad where out > 0:  per row S1 = sum gm, S2 = sum gm xc.  The gate's gradients need only these:
//   dw = sigmoid(w) (1 - sigmoid(w)) (weight / s S2 + bias S1),  db = S1,  dh = (fc2^T (dw, db)) [h > 0],  dq = fc1^T dh
//   dy = gm sigmoid(w) + dq / hw,   dbias = sum dy,   dweight = sum dy xc / s
//   dx = weight / s (dy - dbias / m - xc / s dweight / m)  with m = n hw;  dresidual = gm
// and the channel sums of dy come from S1, S2, dq and the board means, so grad and x are read twice.
//
// What bounds it: memory (the arithmetic is a handful of operations per value).  The plain form reads or writes 7
// activations, the gated one 10, of which 4 and 6 could not be avoided by any form; whether out > 0 is kept as a byte per
// 16 bytes of x.  Statistics are taken about a value of the row (its first), then joined as centred sums in 64 bits: no
// difference of large squares anywhere.
#include <math.h>

#include <type_traits>

#include "train_common.h"

namespace az {

constexpr int NORM_THREADS = 256;
constexpr int GATE_ROWS = 4;                 // boards per workgroup of the gate kernels
constexpr int NORM_MAX_GATED = 1024;         // their LDS: GATE_ROWS * (2 c + hidden) floats

struct NormParams {
    int64_t n;
    int c, hw, hidden, nvec;                 // nvec: 16-byte pieces of a row (hw values, or c with channels last)
    int training;
    uint32_t rows;                           // n * c
    double eps, momentum;
    const float *weight, *bias;
    float *running_mean, *running_var;
    int64_t* num_batches;
    const float *w1, *b1, *w2, *b2;
    // saved
    float *mean, *inv;                       // [c]
    float *board_mean, *gate, *h;            // [n][c], [n][c], [n][hidden] (board_mean: workspace if plain)
    uint8_t* mask;                           // a byte per 16 bytes of x: out > 0
    // forward workspace
    float *m2, *A, *B;                       // [n][c]; A, B per row if gated, per channel if plain
    // backward workspace
    float *s1, *s2, *de, *dh, *dq, *ca, *cb, *cd;   // [n][c] x 2, [n][2c], [n][hidden], [n][c]; per channel
    float* partial;                          // [splits][tiles][TILE_OUT]
    float *dweight, *dbias, *dw1, *db1, *dw2, *db2;
};

__device__ inline float not_below_zero(float v) { return v < 0.f ? 0.f : v; }     // a NaN stays one

__device__ void join_weights(const NormParams& p, int block);

// ---------------------------------------------------------------------------- [n][c][hw]: L lanes to a row
constexpr int ROWS_AT_ONCE = 4;              // rows per group of lanes: that many loads in flight

template <int L>
__device__ inline uint32_t row_of(int k, uint32_t block = blockIdx.x) {
    return (block * ROWS_AT_ONCE + k) * (NORM_THREADS / L) + threadIdx.x / L;
}

template <typename T, int L>
__global__ __launch_bounds__(NORM_THREADS) void k_row_stats(const T* __restrict__ x, const NormParams p) {
    constexpr int V = Pack<T>::V;
    const int lane = threadIdx.x % L;
    float first[ROWS_AT_ONCE], s[ROWS_AT_ONCE], ss[ROWS_AT_ONCE];
#pragma unroll
    for (int k = 0; k < ROWS_AT_ONCE; ++k) {
        const uint32_t row = row_of<L>(k);
        const T* xr = x + (size_t)(row < p.rows ? row : 0) * p.hw;
        first[k] = (float)xr[0];
        s[k] = ss[k] = 0.f;
        for (int j = lane; j < p.nvec; j += L) {
            const int left = p.hw - j * V;
            const auto v = load_pack(xr + j * V, left);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = i < left ? v[i] - first[k] : 0.f;
                s[k] += d;
                ss[k] += d * d;
            }
        }
    }
#pragma unroll
    for (int k = 0; k < ROWS_AT_ONCE; ++k) {
        const uint32_t row = row_of<L>(k);
        const float a = lane_sum<L>(s[k]), b = lane_sum<L>(ss[k]);
        if (lane == 0 && row < p.rows) {
            p.board_mean[row] = first[k] + a / (float)p.hw;
            p.m2[row] = not_below_zero(b - a * a / (float)p.hw);
        }
    }
}

template <typename T, int L, bool GATED>
__global__ __launch_bounds__(NORM_THREADS) void k_row_apply(const T* __restrict__ x, const T* __restrict__ residual,
                                                            T* __restrict__ out, const NormParams p) {
    constexpr int V = Pack<T>::V;
    const int lane = threadIdx.x % L;
#pragma unroll
    for (int k = 0; k < ROWS_AT_ONCE; ++k) {
        const uint32_t row = row_of<L>(k);
        if (row >= p.rows) continue;
        const size_t at = (size_t)row * p.hw;
        const uint32_t q = GATED ? row : row % (uint32_t)p.c;
        const float A = p.A[q], B = p.B[q];
        for (int j = lane; j < p.nvec; j += L) {
            const int left = p.hw - j * V;
            auto v = load_pack(x + at + j * V, left) * A + B;
            if (GATED) v += load_pack(residual + at + j * V, left);
            uint32_t bits = 0;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                bits |= (v[i] > 0.f ? 1u : 0u) << i;
                v[i] = not_below_zero(v[i]);
            }
            store_pack(out + at + j * V, v, left);
            if (p.mask) p.mask[(size_t)row * p.nvec + j] = (uint8_t)bits;
        }
    }
}

template <typename T, int L, bool GATED>
__global__ __launch_bounds__(NORM_THREADS) void k_row_grad_sums(const T* __restrict__ x, const T* __restrict__ grad,
                                                                T* __restrict__ dresidual, const NormParams p) {
    constexpr int V = Pack<T>::V;
    const int lane = threadIdx.x % L;
    float s1[ROWS_AT_ONCE], s2[ROWS_AT_ONCE];
#pragma unroll
    for (int k = 0; k < ROWS_AT_ONCE; ++k) {
        const uint32_t row = row_of<L>(k);
        s1[k] = s2[k] = 0.f;
        if (row >= p.rows) continue;
        const size_t at = (size_t)row * p.hw;
        const float mean = p.mean[row % (uint32_t)p.c];
        for (int j = lane; j < p.nvec; j += L) {
            const int left = p.hw - j * V;
            const auto v = load_pack(x + at + j * V, left);
            auto g = load_pack(grad + at + j * V, left);
            const uint32_t bits = p.mask[(size_t)row * p.nvec + j];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                g[i] = bits >> i & 1 ? g[i] : 0.f;
                s1[k] += g[i];
                s2[k] += g[i] * (v[i] - mean);
            }
            if (GATED) store_pack(dresidual + at + j * V, g, left);
        }
    }
#pragma unroll
    for (int k = 0; k < ROWS_AT_ONCE; ++k) {
        const uint32_t row = row_of<L>(k);
        const float a = lane_sum<L>(s1[k]), b = lane_sum<L>(s2[k]);
        if (lane == 0 && row < p.rows) {
            p.s1[row] = a;
            p.s2[row] = b;
        }
    }
}

// grad: the masked one (dresidual) if gated
template <typename T, int L, bool GATED>
__global__ __launch_bounds__(NORM_THREADS) void k_row_grad_apply(const T* __restrict__ x, const T* __restrict__ grad,
                                                                 T* __restrict__ dx, const NormParams p, uint32_t joins) {
    constexpr int V = Pack<T>::V;
    if (GATED && blockIdx.x < joins) {
        join_weights(p, blockIdx.x);
        return;
    }
    const int lane = threadIdx.x % L;
#pragma unroll
    for (int k = 0; k < ROWS_AT_ONCE; ++k) {
        const uint32_t row = row_of<L>(k, blockIdx.x - joins);
        if (row >= p.rows) continue;
        const size_t at = (size_t)row * p.hw;
        const uint32_t c = row % (uint32_t)p.c;
        const float mean = p.mean[c], b = p.cb[c];
        float a = p.ca[c], d = p.cd[c];
        if (GATED) {
            d += a * p.dq[row] / (float)p.hw;
            a *= p.gate[row];
        }
        for (int j = lane; j < p.nvec; j += L) {
            const int left = p.hw - j * V;
            const auto v = load_pack(x + at + j * V, left);
            auto g = load_pack(grad + at + j * V, left);
            const uint32_t bits = GATED ? 0 : p.mask[(size_t)row * p.nvec + j];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (!GATED) g[i] = bits >> i & 1 ? g[i] : 0.f;
                g[i] = g[i] * a + ((v[i] - mean) * b + d);
            }
            store_pack(dx + at + j * V, g, left);
        }
    }
}

// ---------------------------------------------- [n][hw][c]: a workgroup to a board and a range of channels
// Thread (ty, tx): 16 bytes of channels, every ty-th place of the board; the ty are added through LDS.
struct Lanes {
    int tx, ty, step;          // step: places taken at once
    int j;                     // which 16 bytes of the channels
    bool on;
    int c, left;               // first channel, channels from there on
};

template <typename T>
__device__ inline Lanes lanes_of(const NormParams& p, int wide) {
    Lanes l;
    l.tx = threadIdx.x % wide;
    l.ty = threadIdx.x / wide;
    l.step = NORM_THREADS / wide;
    l.j = blockIdx.y * wide + l.tx;
    l.on = l.ty < l.step && l.j < p.nvec;
    l.c = l.j * Pack<T>::V;
    l.left = p.c - l.c;
    return l;
}

template <int V, typename F>
__device__ inline void add_places(F a, F b, const Lanes& l, int wide, float* out_a, float* out_b, int n_out) {
    __shared__ float red[2][NORM_THREADS * V];
    if (l.ty < l.step) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            red[0][(l.ty * wide + l.tx) * V + i] = a[i];
            red[1][(l.ty * wide + l.tx) * V + i] = b[i];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < wide * V; i += NORM_THREADS) {
        float s = 0.f, ss = 0.f;
        for (int y = 0; y < l.step; ++y) {
            s += red[0][y * wide * V + i];
            ss += red[1][y * wide * V + i];
        }
        if (i < n_out) {
            out_a[i] = s;
            out_b[i] = ss;
        }
    }
}

template <typename T>
__global__ __launch_bounds__(NORM_THREADS) void k_last_stats(const T* __restrict__ x, const NormParams p, int wide) {
    constexpr int V = Pack<T>::V;
    typedef typename Pack<T>::f32 F;
    const Lanes l = lanes_of<T>(p, wide);
    const T* xb = x + (size_t)blockIdx.x * p.hw * p.c;
    F s, ss, first;
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = ss[i] = 0.f;
    if (l.on) {
        first = load_pack(xb + l.c, l.left);
        for (int y = l.ty; y < p.hw; y += l.step) {
            const F d = load_pack(xb + (size_t)y * p.c + l.c, l.left) - first;
            s += d;
            ss += d * d;
        }
    }
    const int c0 = blockIdx.y * wide * V;
    float* mean = p.board_mean + (size_t)blockIdx.x * p.c + c0;
    float* m2 = p.m2 + (size_t)blockIdx.x * p.c + c0;
    const int n_out = p.c - c0;
    add_places<V>(s, ss, l, wide, mean, m2, n_out);
    // the same threads that wrote the sums turn them into the mean and the centred sum
    for (int i = threadIdx.x; i < wide * V && i < n_out; i += NORM_THREADS) {
        const float a = mean[i], b = m2[i];
        mean[i] = (float)xb[c0 + i] + a / (float)p.hw;
        m2[i] = not_below_zero(b - a * a / (float)p.hw);
    }
}

template <typename T, bool GATED>
__global__ __launch_bounds__(NORM_THREADS) void k_last_apply(const T* __restrict__ x, const T* __restrict__ residual,
                                                             T* __restrict__ out, const NormParams p, int wide) {
    constexpr int V = Pack<T>::V;
    typedef typename Pack<T>::f32 F;
    const Lanes l = lanes_of<T>(p, wide);
    if (!l.on) return;
    F A, B;
    const size_t q = (GATED ? (size_t)blockIdx.x * p.c : 0) + l.c;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        A[i] = i < l.left ? p.A[q + i] : 0.f;
        B[i] = i < l.left ? p.B[q + i] : 0.f;
    }
    const size_t board = (size_t)blockIdx.x * p.hw;
    for (int y = l.ty; y < p.hw; y += l.step) {
        const size_t at = (board + y) * p.c + l.c;
        F v = load_pack(x + at, l.left) * A + B;
        if (GATED) v += load_pack(residual + at, l.left);
        uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            bits |= (v[i] > 0.f ? 1u : 0u) << i;
            v[i] = not_below_zero(v[i]);
        }
        store_pack(out + at, v, l.left);
        if (p.mask) p.mask[(board + y) * p.nvec + l.j] = (uint8_t)bits;
    }
}

template <typename T, bool GATED>
__global__ __launch_bounds__(NORM_THREADS) void k_last_grad_sums(const T* __restrict__ x, const T* __restrict__ grad,
                                                                 T* __restrict__ dresidual, const NormParams p, int wide) {
    constexpr int V = Pack<T>::V;
    typedef typename Pack<T>::f32 F;
    const Lanes l = lanes_of<T>(p, wide);
    F s1, s2, mean;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        s1[i] = s2[i] = 0.f;
        mean[i] = l.on && i < l.left ? p.mean[l.c + i] : 0.f;
    }
    const size_t board = (size_t)blockIdx.x * p.hw;
    if (l.on)
        for (int y = l.ty; y < p.hw; y += l.step) {
            const size_t at = (board + y) * p.c + l.c;
            const F v = load_pack(x + at, l.left);
            F g = load_pack(grad + at, l.left);
            const uint32_t bits = p.mask[(board + y) * p.nvec + l.j];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                g[i] = bits >> i & 1 ? g[i] : 0.f;
                s1[i] += g[i];
                s2[i] += g[i] * (v[i] - mean[i]);
            }
            if (GATED) store_pack(dresidual + at, g, l.left);
        }
    const int c0 = blockIdx.y * wide * V;
    add_places<V>(s1, s2, l, wide, p.s1 + (size_t)blockIdx.x * p.c + c0, p.s2 + (size_t)blockIdx.x * p.c + c0, p.c - c0);
}

template <typename T, bool GATED>
__global__ __launch_bounds__(NORM_THREADS) void k_last_grad_apply(const T* __restrict__ x, const T* __restrict__ grad,
                                                                  T* __restrict__ dx, const NormParams p, int wide, uint32_t joins) {
    constexpr int V = Pack<T>::V;
    typedef typename Pack<T>::f32 F;
    if (GATED && blockIdx.x < joins) {
        if (blockIdx.y == 0) join_weights(p, blockIdx.x);
        return;
    }
    const uint32_t n = blockIdx.x - joins;
    const Lanes l = lanes_of<T>(p, wide);
    if (!l.on) return;
    F mean, a, b, d;
    const size_t row = (size_t)n * p.c + l.c;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = i < l.left ? l.c + i : 0;
        mean[i] = p.mean[c];
        a[i] = p.ca[c];
        b[i] = p.cb[c];
        d[i] = p.cd[c];
        if (GATED && i < l.left) {
            d[i] += a[i] * p.dq[row + i] / (float)p.hw;
            a[i] *= p.gate[row + i];
        }
    }
    const size_t board = (size_t)n * p.hw;
    for (int y = l.ty; y < p.hw; y += l.step) {
        const size_t at = (board + y) * p.c + l.c;
        const F v = load_pack(x + at, l.left);
        F g = load_pack(grad + at, l.left);
        const uint32_t bits = GATED ? 0 : p.mask[(board + y) * p.nvec + l.j];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (!GATED) g[i] = bits >> i & 1 ? g[i] : 0.f;
            g[i] = g[i] * a[i] + ((v[i] - mean[i]) * b[i] + d[i]);
        }
        store_pack(dx + at, g, l.left);
    }
}

// ------------------------------------------------------------------- per channel: sums over the boards in 64 bits
constexpr int CHANNELS = 4, BOARDS = 128;     // a workgroup: 4 neighbouring channels, 128 boards at a time
constexpr int IN_FLIGHT = 8;                  // boards whose loads a thread has under way

template <int K>
__device__ inline void add_boards(double (&v)[K]) {
    __shared__ double red[BOARDS][CHANNELS][K];
    const int ch = threadIdx.x % CHANNELS, b = threadIdx.x / CHANNELS;
#pragma unroll
    for (int k = 0; k < K; ++k) red[b][ch][k] = v[k];
    for (int half = BOARDS / 2; half; half >>= 1) {
        __syncthreads();
        if (b < half)
#pragma unroll
            for (int k = 0; k < K; ++k) red[b][ch][k] += red[b + half][ch][k];
    }
    if (b == 0)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = red[0][ch][k];
}

__global__ __launch_bounds__(CHANNELS * BOARDS) void k_channel_stats(const NormParams p) {
    const int c = blockIdx.x * CHANNELS + threadIdx.x % CHANNELS, b = threadIdx.x / CHANNELS;
    double v[3] = {0, 0, 0};          // sum of board means, of their squares, of centred sums
    if (p.training) {
        if (c < p.c)
            for (int64_t i = b; i < p.n; i += BOARDS * IN_FLIGHT) {
                float mean[IN_FLIGHT], m2[IN_FLIGHT];
#pragma unroll
                for (int u = 0; u < IN_FLIGHT; ++u) {
                    const int64_t iu = i + u * BOARDS, row = (iu < p.n ? iu : i) * p.c + c;
                    mean[u] = p.board_mean[row];
                    m2[u] = p.m2[row];
                }
#pragma unroll
                for (int u = 0; u < IN_FLIGHT; ++u)
                    if (i + u * BOARDS < p.n) {
                        const double m = mean[u];
                        v[0] += m;
                        v[1] += m * m;
                        v[2] += m2[u];
                    }
            }
        add_boards(v);
    }
    if (b == 0 && c < p.c) {
        double mean, var;
        if (p.training) {
            const double count = (double)p.n * p.hw;
            mean = v[0] / p.n;
            var = (v[2] + p.hw * (v[1] - p.n * mean * mean)) / count;
            if (var < 0.0) var = 0.0;          // a NaN stays one
            if (p.running_mean) p.running_mean[c] = (float)((1.0 - p.momentum) * p.running_mean[c] + p.momentum * mean);
            if (p.running_var) p.running_var[c] = (float)((1.0 - p.momentum) * p.running_var[c] + p.momentum * var * count / (count - 1.0));
        } else {
            mean = p.running_mean[c];
            var = p.running_var[c];
        }
        const float inv = (float)(1.0 / sqrt(var + p.eps)), m = (float)mean;
        p.mean[c] = m;
        p.inv[c] = inv;
        if (!p.hidden) {
            p.A[c] = p.weight[c] * inv;
            p.B[c] = p.bias[c] - p.weight[c] * inv * m;
        }
    }
    if (p.num_batches && p.training && blockIdx.x == 0 && threadIdx.x == 0) *p.num_batches += 1;
}

// dy's channel sums, and with them what the last pass needs: dx = ca gm (gate) + (x - mean) cb + cd (+ ca dq / hw)
__device__ inline void channel_grads(const NormParams& p, int block) {
    const int c = block * CHANNELS + threadIdx.x % CHANNELS, b = threadIdx.x / CHANNELS;
    double v[2] = {0, 0};
    if (c < p.c) {
        const float mean = p.mean[c];
        for (int64_t i = b; i < p.n; i += BOARDS * IN_FLIGHT) {
            float s1[IN_FLIGHT], s2[IN_FLIGHT], gate[IN_FLIGHT], dq[IN_FLIGHT], bm[IN_FLIGHT];
#pragma unroll
            for (int u = 0; u < IN_FLIGHT; ++u) {
                const int64_t iu = i + u * BOARDS, row = (iu < p.n ? iu : i) * p.c + c;
                s1[u] = p.s1[row];
                s2[u] = p.s2[row];
                if (p.hidden) {
                    gate[u] = p.gate[row];
                    dq[u] = p.dq[row];
                    bm[u] = p.board_mean[row];
                }
            }
#pragma unroll
            for (int u = 0; u < IN_FLIGHT; ++u)
                if (i + u * BOARDS < p.n) {
                    if (p.hidden) {
                        s1[u] = gate[u] * s1[u] + dq[u];
                        s2[u] = gate[u] * s2[u] + dq[u] * (bm[u] - mean);
                    }
                    v[0] += s1[u];
                    v[1] += s2[u];
                }
        }
    }
    add_boards(v);
    if (b == 0 && c < p.c) {
        const float inv = p.inv[c], a = p.weight[c] * inv;
        const double count = (double)p.n * p.hw;
        p.dbias[c] = (float)v[0];
        p.dweight[c] = (float)(v[1] * inv);
        p.ca[c] = a;
        p.cb[c] = p.training ? (float)(-a * inv * inv * (v[1] / count)) : 0.f;
        p.cd[c] = p.training ? (float)(-a * (v[0] / count)) : 0.f;
    }
}

// --------------------------------------------------------------------------------------------- the gate
__global__ __launch_bounds__(256) void k_gate_forward(const NormParams p) {
    extern __shared__ float lds[];
    float* q = lds;                                  // [GATE_ROWS][c]
    float* h = lds + GATE_ROWS * p.c;                // [GATE_ROWS][hidden]
    const int64_t n0 = (int64_t)blockIdx.x * GATE_ROWS;
    const int rows = (int)(p.n - n0 < GATE_ROWS ? p.n - n0 : GATE_ROWS);
    for (int i = threadIdx.x; i < GATE_ROWS * p.c; i += 256) {
        const int c = i % p.c;
        q[i] = i / p.c < rows ? (p.board_mean[n0 * p.c + i] - p.mean[c]) * (p.weight[c] * p.inv[c]) + p.bias[c] : 0.f;
    }
    __syncthreads();
    // four lanes to a hidden unit of a board
    for (int o = threadIdx.x / 4; o < GATE_ROWS * p.hidden; o += 64) {
        const int r = o / p.hidden, k = o % p.hidden;
        float s = 0.f;
        for (int c = threadIdx.x % 4; c < p.c; c += 4) s += p.w1[(size_t)k * p.c + c] * q[r * p.c + c];
        s = lane_sum<4>(s);
        if (threadIdx.x % 4 == 0) {
            const float on = not_below_zero(s + p.b1[k]);
            h[o] = on;
            if (r < rows) p.h[(n0 + r) * p.hidden + k] = on;
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < p.c; c += 256) {
        float w[GATE_ROWS], b[GATE_ROWS];
#pragma unroll
        for (int r = 0; r < GATE_ROWS; ++r) {
            w[r] = p.b2[c];
            b[r] = p.b2[p.c + c];
        }
        for (int k = 0; k < p.hidden; ++k) {
            const float ww = p.w2[(size_t)c * p.hidden + k], wb = p.w2[(size_t)(p.c + c) * p.hidden + k];
#pragma unroll
            for (int r = 0; r < GATE_ROWS; ++r) {
                w[r] += ww * h[r * p.hidden + k];
                b[r] += wb * h[r * p.hidden + k];
            }
        }
        const float scale = p.weight[c] * p.inv[c], shift = p.bias[c] - scale * p.mean[c];
#pragma unroll
        for (int r = 0; r < GATE_ROWS; ++r)
            if (r < rows) {
                const int64_t row = (n0 + r) * p.c + c;
                const float gate = 1.f / (1.f + expf(-w[r]));
                p.gate[row] = gate;
                p.A[row] = scale * gate;
                p.B[row] = shift * gate + b[r];
            }
    }
}

__global__ __launch_bounds__(256) void k_gate_backward(const NormParams p) {
    extern __shared__ float lds[];
    float* de = lds;                                 // [GATE_ROWS][2c]
    float* dh = lds + GATE_ROWS * 2 * p.c;           // [GATE_ROWS][hidden]
    const int64_t n0 = (int64_t)blockIdx.x * GATE_ROWS;
    const int rows = (int)(p.n - n0 < GATE_ROWS ? p.n - n0 : GATE_ROWS);
    for (int i = threadIdx.x; i < GATE_ROWS * p.c; i += 256) {
        const int r = i / p.c, c = i % p.c;
        float w = 0.f, b = 0.f;
        if (r < rows) {
            const int64_t row = (n0 + r) * p.c + c;
            const float gate = p.gate[row];
            b = p.s1[row];
            w = gate * (1.f - gate) * (p.weight[c] * p.inv[c] * p.s2[row] + p.bias[c] * b);
            p.de[(n0 + r) * 2 * p.c + c] = w;
            p.de[(n0 + r) * 2 * p.c + p.c + c] = b;
        }
        de[r * 2 * p.c + c] = w;
        de[r * 2 * p.c + p.c + c] = b;
    }
    __syncthreads();
    // a wavefront to a hidden unit: its column of fc2 against the four boards
    for (int k = threadIdx.x / 64; k < p.hidden; k += 4) {
        float s[GATE_ROWS] = {};
        for (int j = threadIdx.x % 64; j < 2 * p.c; j += 64) {
            const float w = p.w2[(size_t)j * p.hidden + k];
#pragma unroll
            for (int r = 0; r < GATE_ROWS; ++r) s[r] += w * de[r * 2 * p.c + j];
        }
#pragma unroll
        for (int r = 0; r < GATE_ROWS; ++r) {
            s[r] = lane_sum<64>(s[r]);
            if (r >= rows || !(p.h[(n0 + (r < rows ? r : 0)) * p.hidden + k] > 0.f)) s[r] = 0.f;
            if (threadIdx.x % 64 == 0) {
                dh[r * p.hidden + k] = s[r];
                if (r < rows) p.dh[(n0 + r) * p.hidden + k] = s[r];
            }
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < p.c; c += 256) {
        float s[GATE_ROWS] = {};
        for (int k = 0; k < p.hidden; ++k) {
            const float w = p.w1[(size_t)k * p.c + c];
#pragma unroll
            for (int r = 0; r < GATE_ROWS; ++r) s[r] += w * dh[r * p.hidden + k];
        }
#pragma unroll
        for (int r = 0; r < GATE_ROWS; ++r)
            if (r < rows) p.dq[(n0 + r) * p.c + c] = s[r];
    }
}

// Gradients of the gate's weights: sums over the boards of outer products, as 32 x 32 tiles.  A workgroup takes one tile and
// one of `splits` ranges of boards, each of its wavefronts every eighth board, a lane 4 x 4 of the tile, four boards' loads
// in flight.  The bias is the sum of the left factor.  The partial tiles go to the workspace; the last pass's first
// workgroups add them in order, beside its own work.
// (One workgroup per tile over all boards, one board in flight, took 62 us at 1024 x 128 and 230 us at 4096 x 256: four times
// the pass over the activations that follows.)
constexpr int TILE = 32, TILE_WAVES = CHANNELS * BOARDS / 64, TILE_BOARDS = 4, TILE_OUT = TILE * TILE + TILE;

struct TileShape {
    int m, k, across, tiles;                                         // [m][k] in `tiles` tiles, `across` to a row
};

__host__ __device__ inline TileShape tile_shape(int m, int k) {
    const int across = (k + TILE - 1) / TILE;
    return {m, k, across, (m + TILE - 1) / TILE * across};
}

__host__ __device__ inline int weight_tiles(const NormParams& p) { return tile_shape(2 * p.c, p.hidden).tiles + tile_shape(p.hidden, p.c).tiles; }

// Ranges of at least 64 boards (two rounds of a wavefront), and no more than fill the chip a few times.
__host__ __device__ inline int weight_splits(const NormParams& p) {
    const int64_t most = (p.n + 63) / 64, enough = 2048 / weight_tiles(p);
    return (int)(enough < 1 ? 1 : most < enough ? most : enough);
}

__device__ inline void weight_tile(const NormParams& p, int job) {
    __shared__ float lds[TILE_WAVES][TILE_OUT];
    const int tiles = weight_tiles(p), splits = weight_splits(p), split = job / tiles;
    int tile = job % tiles;
    const TileShape fc2 = tile_shape(2 * p.c, p.hidden), fc1 = tile_shape(p.hidden, p.c);
    const bool second = tile < fc2.tiles;
    const TileShape t = second ? fc2 : fc1;
    if (!second) tile -= fc2.tiles;
    const int i0 = tile / t.across * TILE, j0 = tile % t.across * TILE;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = i0 + lane / 8 * 4, lj = j0 + lane % 8 * 4;
    const float *left = second ? p.de : p.dh, *right = second ? p.h : p.board_mean;
    f32x4 acc[4], bias, scale, shift;                                // fc1's right factor: q = mean * scale + shift
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        acc[j] = 0.f;
        bias[j] = 0.f;
        const int c = lj + j < t.k ? lj + j : 0;
        scale[j] = second ? 1.f : p.weight[c] * p.inv[c];
        shift[j] = second ? 0.f : p.bias[c] - scale[j] * p.mean[c];
    }
    const int64_t from = p.n * split / splits, to = p.n * (split + 1) / splits;
    for (int64_t n = from + wave; n < to; n += TILE_WAVES * TILE_BOARDS) {
        f32x4 a[TILE_BOARDS], b[TILE_BOARDS];
#pragma unroll
        for (int u = 0; u < TILE_BOARDS; ++u) {
            const int64_t nu = n + u * TILE_WAVES;
            const bool in = nu < to;
            a[u] = load_pack(left + (in ? nu : n) * t.m + li, in ? t.m - li : 0);
            b[u] = load_pack(right + (in ? nu : n) * t.k + lj, t.k - lj);
        }
#pragma unroll
        for (int u = 0; u < TILE_BOARDS; ++u) {
            const f32x4 q = b[u] * scale + shift;
            bias += a[u];
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] += a[u][i] * q;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) *(f32x4*)&lds[wave][(lane / 8 * 4 + i) * TILE + lane % 8 * 4] = acc[i];
    if (lane % 8 == 0) *(f32x4*)&lds[wave][TILE * TILE + lane / 8 * 4] = bias;
    __syncthreads();
    float* out = p.partial + ((size_t)split * tiles + job % tiles) * TILE_OUT;
    for (int o = threadIdx.x; o < TILE_OUT; o += TILE_WAVES * 64) {
        float s = lds[0][o];
        for (int w = 1; w < TILE_WAVES; ++w) s += lds[w][o];
        out[o] = s;
    }
}

// One output per thread: the partial tiles in order.
__device__ void join_weights(const NormParams& p, int block) {
    const int tiles = weight_tiles(p), splits = weight_splits(p);
    const int o = block * NORM_THREADS + threadIdx.x;
    if (o >= tiles * TILE_OUT) return;
    float s = 0.f;
    for (int i = 0; i < splits; ++i) s += p.partial[(size_t)i * tiles * TILE_OUT + o];
    int tile = o / TILE_OUT;
    const int at = o % TILE_OUT;
    const TileShape fc2 = tile_shape(2 * p.c, p.hidden), fc1 = tile_shape(p.hidden, p.c);
    const bool second = tile < fc2.tiles;
    const TileShape t = second ? fc2 : fc1;
    if (!second) tile -= fc2.tiles;
    const int i0 = tile / t.across * TILE, j0 = tile % t.across * TILE;
    if (at < TILE * TILE) {
        const int i = i0 + at / TILE, j = j0 + at % TILE;
        if (i < t.m && j < t.k) (second ? p.dw2 : p.dw1)[(size_t)i * t.k + j] = s;
    } else {
        const int i = i0 + at - TILE * TILE;
        if (i < t.m && j0 == 0) (second ? p.db2 : p.db1)[i] = s;
    }
}

static int join_blocks(const NormParams& p) { return p.hidden ? (weight_tiles(p) * TILE_OUT + NORM_THREADS - 1) / NORM_THREADS : 0; }

__global__ __launch_bounds__(CHANNELS * BOARDS) void k_param_grads(const NormParams p, int channel_blocks) {
    if ((int)blockIdx.x < channel_blocks) channel_grads(p, blockIdx.x);
    else weight_tile(p, (int)blockIdx.x - channel_blocks);
}

// ---------------------------------------------------------------------------------------------- host side
// Lanes to a row: a piece of 16 bytes each, as many as the row has, up to 16 (a longer row takes several rounds).
template <typename F>
static void with_lanes(int nvec, F&& f) {
    if (nvec <= 4) f(std::integral_constant<int, 4>());
    else if (nvec <= 8) f(std::integral_constant<int, 8>());
    else f(std::integral_constant<int, 16>());
}

template <typename T>
static int norm_forward(const NormParams& p, bool last, const void* x, const void* residual, void* out, hipStream_t s) {
    const T *xt = (const T*)x, *rt = (const T*)residual;
    T* ot = (T*)out;
    const bool need_rows = p.training || p.hidden;
    const int wide = p.nvec < 64 ? p.nvec : 64;
    const dim3 boards((uint32_t)p.n, (p.nvec + wide - 1) / wide), block(NORM_THREADS);
    if (need_rows) {
        if (last) hipLaunchKernelGGL((k_last_stats<T>), boards, block, 0, s, xt, p, wide);
        else with_lanes(p.nvec, [&](auto L) {
            const uint32_t per = NORM_THREADS / L * ROWS_AT_ONCE;
            hipLaunchKernelGGL((k_row_stats<T, decltype(L)::value>), dim3((p.rows + per - 1) / per), block, 0, s, xt, p);
        });
        AZ_HIP(hipGetLastError());
    }
    hipLaunchKernelGGL(k_channel_stats, dim3((p.c + CHANNELS - 1) / CHANNELS), dim3(CHANNELS * BOARDS), 0, s, p);
    AZ_HIP(hipGetLastError());
    if (p.hidden) {
        hipLaunchKernelGGL(k_gate_forward, dim3((uint32_t)((p.n + GATE_ROWS - 1) / GATE_ROWS)), dim3(256),
                           sizeof(float) * GATE_ROWS * (p.c + p.hidden), s, p);
        AZ_HIP(hipGetLastError());
    }
    if (last) {
        if (p.hidden) hipLaunchKernelGGL((k_last_apply<T, true>), boards, block, 0, s, xt, rt, ot, p, wide);
        else hipLaunchKernelGGL((k_last_apply<T, false>), boards, block, 0, s, xt, rt, ot, p, wide);
    } else {
        with_lanes(p.nvec, [&](auto L) {
            constexpr int N = decltype(L)::value;
            const uint32_t per = NORM_THREADS / N * ROWS_AT_ONCE;
            const dim3 grid((p.rows + per - 1) / per);
            if (p.hidden) hipLaunchKernelGGL((k_row_apply<T, N, true>), grid, block, 0, s, xt, rt, ot, p);
            else hipLaunchKernelGGL((k_row_apply<T, N, false>), grid, block, 0, s, xt, rt, ot, p);
        });
    }
    AZ_HIP(hipGetLastError());
    return AZ_OK;
}

template <typename T>
static int norm_backward(const NormParams& p, bool last, const void* x, const void* grad, void* dx, void* dresidual, hipStream_t s) {
    const T *xt = (const T*)x, *gt = (const T*)grad;
    T *dt = (T*)dx, *rt = (T*)dresidual;
    const int wide = p.nvec < 64 ? p.nvec : 64;
    const dim3 boards((uint32_t)p.n, (p.nvec + wide - 1) / wide), block(NORM_THREADS);
    if (last) {
        if (p.hidden) hipLaunchKernelGGL((k_last_grad_sums<T, true>), boards, block, 0, s, xt, gt, rt, p, wide);
        else hipLaunchKernelGGL((k_last_grad_sums<T, false>), boards, block, 0, s, xt, gt, rt, p, wide);
    } else {
        with_lanes(p.nvec, [&](auto L) {
            constexpr int N = decltype(L)::value;
            const uint32_t per = NORM_THREADS / N * ROWS_AT_ONCE;
            const dim3 grid((p.rows + per - 1) / per);
            if (p.hidden) hipLaunchKernelGGL((k_row_grad_sums<T, N, true>), grid, block, 0, s, xt, gt, rt, p);
            else hipLaunchKernelGGL((k_row_grad_sums<T, N, false>), grid, block, 0, s, xt, gt, rt, p);
        });
    }
    AZ_HIP(hipGetLastError());
    if (p.hidden) {
        hipLaunchKernelGGL(k_gate_backward, dim3((uint32_t)((p.n + GATE_ROWS - 1) / GATE_ROWS)), dim3(256),
                           sizeof(float) * GATE_ROWS * (2 * p.c + p.hidden), s, p);
        AZ_HIP(hipGetLastError());
    }
    const int cb = (p.c + CHANNELS - 1) / CHANNELS;
    hipLaunchKernelGGL(k_param_grads, dim3(cb + (p.hidden ? weight_tiles(p) * weight_splits(p) : 0)), dim3(CHANNELS * BOARDS), 0, s, p, cb);
    AZ_HIP(hipGetLastError());
    const T* mt = p.hidden ? rt : gt;
    const uint32_t joins = (uint32_t)join_blocks(p);
    if (last) {
        const dim3 grid(boards.x + joins, boards.y);
        if (p.hidden) hipLaunchKernelGGL((k_last_grad_apply<T, true>), grid, block, 0, s, xt, mt, dt, p, wide, joins);
        else hipLaunchKernelGGL((k_last_grad_apply<T, false>), grid, block, 0, s, xt, mt, dt, p, wide, joins);
    } else {
        with_lanes(p.nvec, [&](auto L) {
            constexpr int N = decltype(L)::value;
            const uint32_t per = NORM_THREADS / N * ROWS_AT_ONCE;
            const dim3 grid((p.rows + per - 1) / per + joins);
            if (p.hidden) hipLaunchKernelGGL((k_row_grad_apply<T, N, true>), grid, block, 0, s, xt, mt, dt, p, joins);
            else hipLaunchKernelGGL((k_row_grad_apply<T, N, false>), grid, block, 0, s, xt, mt, dt, p, joins);
        });
    }
    AZ_HIP(hipGetLastError());
    return AZ_OK;
}

static size_t round16(size_t bytes) { return (bytes + 15) / 16 * 16; }

// Hands out pieces of a buffer, 16-byte aligned.
struct Carver {
    char* base;
    size_t used;
    template <typename T> T* take(size_t count) {
        T* r = base ? (T*)(base + used) : nullptr;
        used += round16(count * sizeof(T));
        return r;
    }
};

static int norm_params(const az_norm_args* a, NormParams* p, int64_t sizes[3]) {
    AZ_CHECK_ARG(a, "norm: null arguments");
    AZ_CHECK_ARG(a->dtype == AZ_F32 || a->dtype == AZ_BF16 || a->dtype == AZ_F16, "norm: unknown type %d", a->dtype);
    AZ_CHECK_ARG(a->n >= 1 && a->c >= 1 && a->hw >= 1 && a->hw <= 1 << 24 && a->n <= 0x7FFFFFFF && a->n * a->c <= 0x7FFFFFFF,
                 "norm: sizes %lld x %d x %d out of range", (long long)a->n, a->c, a->hw);
    AZ_CHECK_ARG(!a->training || a->n * a->hw >= 2, "norm: the batch's statistics need two values per channel");
    AZ_CHECK_ARG(a->hidden >= 0 && (a->hidden == 0 || (a->c <= NORM_MAX_GATED && a->hidden <= NORM_MAX_GATED)),
                 "norm: a gate takes up to %d channels and hidden units (got %d, %d)", NORM_MAX_GATED, a->c, a->hidden);
    const int V = a->dtype == AZ_F32 ? 4 : 8;
    const size_t rows = (size_t)a->n * a->c, hidden = (size_t)a->n * a->hidden;
    p->n = a->n;
    p->c = a->c;
    p->hw = a->hw;
    p->hidden = a->hidden;
    p->nvec = ((a->channels_last ? a->c : a->hw) + V - 1) / V;
    p->training = a->training != 0;
    p->rows = (uint32_t)rows;
    p->eps = a->eps;
    p->momentum = a->momentum;
    p->weight = a->weight_dev;
    p->bias = a->bias_dev;
    p->running_mean = a->running_mean_dev;
    p->running_var = a->running_var_dev;
    p->num_batches = a->num_batches_dev;
    p->w1 = a->fc1_weight_dev;
    p->b1 = a->fc1_bias_dev;
    p->w2 = a->fc2_weight_dev;
    p->b2 = a->fc2_bias_dev;
    p->dweight = a->dweight_dev;
    p->dbias = a->dbias_dev;
    p->dw1 = a->dfc1_weight_dev;
    p->db1 = a->dfc1_bias_dev;
    p->dw2 = a->dfc2_weight_dev;
    p->db2 = a->dfc2_bias_dev;
    Carver saved = {(char*)a->saved_dev, 0}, fwd = {(char*)a->workspace_dev, 0}, bwd = {(char*)a->workspace_dev, 0};
    p->mean = saved.take<float>(a->c);
    p->inv = saved.take<float>(a->c);
    if (a->hidden) {
        p->board_mean = saved.take<float>(rows);
        p->gate = saved.take<float>(rows);
        p->h = saved.take<float>(hidden);
    } else {
        p->board_mean = fwd.take<float>(rows);
        p->gate = p->h = nullptr;
    }
    p->mask = saved.take<uint8_t>((size_t)p->nvec * (a->channels_last ? (size_t)a->n * a->hw : rows));
    p->m2 = fwd.take<float>(rows);
    p->A = fwd.take<float>(a->hidden ? rows : a->c);
    p->B = fwd.take<float>(a->hidden ? rows : a->c);
    p->s1 = bwd.take<float>(rows);
    p->s2 = bwd.take<float>(rows);
    p->ca = bwd.take<float>(a->c);
    p->cb = bwd.take<float>(a->c);
    p->cd = bwd.take<float>(a->c);
    p->de = p->dh = p->dq = p->partial = nullptr;
    if (a->hidden) {
        p->de = bwd.take<float>(2 * rows);
        p->dh = bwd.take<float>(hidden);
        p->dq = bwd.take<float>(rows);
        p->partial = bwd.take<float>((size_t)weight_tiles(*p) * weight_splits(*p) * TILE_OUT);
    }
    if (sizes) {
        sizes[0] = (int64_t)saved.used;
        sizes[1] = (int64_t)fwd.used;
        sizes[2] = (int64_t)bwd.used;
    }
    return AZ_OK;
}

static int norm_check(const az_norm_args* a) {
    AZ_CHECK_ARG(a->x_dev && a->weight_dev && a->bias_dev && a->saved_dev && a->workspace_dev, "norm: null argument");
    AZ_CHECK_ARG((uintptr_t)a->saved_dev % 16 == 0 && (uintptr_t)a->workspace_dev % 16 == 0, "norm: buffers must be 16-byte aligned");
    AZ_CHECK_ARG(!a->hidden || (a->fc1_weight_dev && a->fc1_bias_dev && a->fc2_weight_dev && a->fc2_bias_dev), "norm: null gate weights");
    return AZ_OK;
}

}  // namespace az

using namespace az;

extern "C" int az_norm_sizes(const az_norm_args* a, int64_t sizes_host[3]) {
    AZ_CHECK_ARG(sizes_host, "az_norm_sizes: null output");
    NormParams p;
    return norm_params(a, &p, sizes_host);
}

extern "C" int az_norm_forward(const az_norm_args* a, void* stream) {
    NormParams p;
    int rc = norm_params(a, &p, nullptr);
    if (rc == AZ_OK) rc = norm_check(a);
    if (rc != AZ_OK) return rc;
    AZ_CHECK_ARG(a->out_dev && (!a->hidden || a->residual_dev), "az_norm_forward: null argument");
    AZ_CHECK_ARG(a->training || (a->running_mean_dev && a->running_var_dev), "az_norm_forward: evaluation without running statistics");
    const bool last = a->channels_last != 0;
    switch (a->dtype) {
        case AZ_F32: return norm_forward<float>(p, last, a->x_dev, a->residual_dev, a->out_dev, (hipStream_t)stream);
        case AZ_BF16: return norm_forward<__bf16>(p, last, a->x_dev, a->residual_dev, a->out_dev, (hipStream_t)stream);
        default: return norm_forward<_Float16>(p, last, a->x_dev, a->residual_dev, a->out_dev, (hipStream_t)stream);
    }
}

extern "C" int az_norm_backward(const az_norm_args* a, void* stream) {
    NormParams p;
    int rc = norm_params(a, &p, nullptr);
    if (rc == AZ_OK) rc = norm_check(a);
    if (rc != AZ_OK) return rc;
    AZ_CHECK_ARG(a->grad_dev && a->dx_dev && a->dweight_dev && a->dbias_dev, "az_norm_backward: null argument");
    AZ_CHECK_ARG(!a->hidden || (a->dresidual_dev && a->dfc1_weight_dev && a->dfc1_bias_dev && a->dfc2_weight_dev && a->dfc2_bias_dev),
                 "az_norm_backward: null gate gradient");
    const bool last = a->channels_last != 0;
    switch (a->dtype) {
        case AZ_F32: return norm_backward<float>(p, last, a->x_dev, a->grad_dev, a->dx_dev, a->dresidual_dev, (hipStream_t)stream);
        case AZ_BF16: return norm_backward<__bf16>(p, last, a->x_dev, a->grad_dev, a->dx_dev, a->dresidual_dev, (hipStream_t)stream);
        default: return norm_backward<_Float16>(p, last, a->x_dev, a->grad_dev, a->dx_dev, a->dresidual_dev, (hipStream_t)stream);
    }
}
