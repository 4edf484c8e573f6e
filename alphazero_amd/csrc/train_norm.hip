// Batch normalisation with ReLU, and the end of a squeeze-excitation residual block, forward and backward.
//
// Mathematics, for a convolution's output x (n boards, c channels, hw places), mu and 1/s from the batch (or the running
// statistics), xc = x - mu:
//   y = weight xc / s + bias                                          plain:  out = relu(y)
//   q = mean_hw y,  h = relu(fc1 q + b1),  (w, b) = fc2 h + b2        gated:  out = relu(y sigmoid(w) + b + residual)
// Forward: one pass over x takes the mean and the centred sum of squares of every board and channel ("row"); from these
// come the batch's statistics and the squeeze q, so x is read once more only, for out = relu(A xc + B (+ residual)) with
// A, B per row (gated) or per channel (plain): xc first, so that what mu and x have in common is gone before anything is rounded.
// Backward, with gm = grad where out > 0 (or out is a NaN):  per row S1 = sum gm, S2 = sum gm xc.  The gate's gradients need only these:
//   dw = sigmoid(w) (1 - sigmoid(w)) (weight / s S2 + bias S1),  db = S1,  dh = (fc2^T (dw, db)) [h > 0],  dq = fc1^T dh
//   dy = gm sigmoid(w) + dq / hw,   dbias = sum dy,   dweight = sum dy xc / s
//   dx = weight / s (dy - dbias / m - xc / s dweight / m)  with m = n hw;  dresidual = gm
// and the channel sums of dy come from S1, S2, dq and the board means, so grad and x are read twice.
//
// What bounds it: memory (the arithmetic is a handful of operations per value).  Both directions together, the plain form reads
// or writes 8 activations and the gated one 10: x and the gradient are needed again once the batch's sums are known.  A
// plain norm whose channels fit a workgroup's registers takes 5, each tensor once a direction (4 and 6 are the different tensors
// there are; x belongs to two calls).  The passes keep whether out > 0 as a byte per 16 bytes of x.
// Statistics are means and centred sums of a row (about its own mean, or joined piece by piece in long rows and
// channels-last), so that no square of a distance from somewhere else is taken off again; over the chunks of boards they are
// joined in 64 bits, where the squares of the means may be subtracted.
// Measured, forward and backward: at 4096 x 256 x 64 in bfloat16 (134 MB a tensor) 296 us, of which the four passes over
// activations take 240 (1.34 GB: 5.6 TB/s; a copy of 1 GiB reaches 5.1) and the gate and the channel sums 57; at
// 1024 x 128 x 64 in float32 83 us (61 and 22); a plain norm at 1024 x 128 x 64 in bfloat16 31 us.
#include <math.h>

#include <type_traits>

#include "train_common.h"

namespace az {

constexpr int NORM_THREADS = 256;
constexpr int GATE_ROWS = 4;                 // boards per workgroup of the gate kernels
constexpr int NORM_MAX_GATED = 1024;         // their LDS: 16 (3 c + hidden) bytes forward, 16 (2 c + hidden + 1024) backward: 64 KB

struct NormParams {
    int64_t n;
    int c, hw, hidden, nvec;                 // nvec: 16-byte pieces of a row (hw values, or c with channels last)
    int training, by_channel;
    double eps, momentum, per_count, to_sample;      // the values of a channel: one by their number, number / (number - 1)
    const float *weight, *bias;
    float *running_mean, *running_var;
    int64_t* num_batches;
    const float *w1, *b1, *w2, *b2;
    // saved
    float *mean, *inv;                       // [c]
    float *board_mean, *gate, *h;            // gated: [n][c], [n][c], [n][hidden]
    uint8_t* mask;                           // a byte per 16 bytes of x: out > 0
    // partial sums over chunks of boards, [chunks][c]: means and centred sums forward, dy's sums backward
    float *part_a, *part_b;
    int64_t chunks;
    int chunk_boards, abreast;
    // forward workspace
    float *A, *B;                            // per row if gated, per channel if plain
    // backward workspace
    float *s1, *s2, *de, *dh, *dq, *ca, *cb, *cd;   // gated: [n][c] x 2, [n][2c], [n][hidden], [n][c]; per channel
    float* partial;                          // [splits][tiles][TILE_OUT]
    float *dweight, *dbias, *dw1, *db1, *dw2, *db2;
};

__device__ inline float not_below_zero(float v) { return v < 0.f ? 0.f : v; }     // a NaN stays one

__device__ void join_weights(const NormParams& p, int block);

// The boards whose sums chunk i holds: p.chunk_boards of them, p.abreast apart, fewer at the end.
__device__ inline uint32_t boards_in_chunk(const NormParams& p, uint32_t i) {
    const uint32_t n = (uint32_t)p.n, side = (uint32_t)p.abreast, most = (uint32_t)p.chunk_boards;
    const uint32_t beside = side == 1 ? 0 : i % side, first = (i - beside) * most + beside;
    const uint32_t k = first >= n ? 0 : side == 1 ? n - first : (n - 1 - first) / side + 1;
    return k < most ? k : most;
}

// The second pass over the activations begins where the first one ended: what was touched last is still in the last-level
// cache.  Workgroups go to the eight dies in turn, so the order is turned round in eights: a workgroup finds what its
// die's own L2 holds of the first pass.  (At 4096 x 256 in bfloat16, 134 MB a tensor: the two second passes 142 us in the
// same order, 136 in reverse; reversed without the eights 1024 x 128, which the L2s hold, loses 10 %.)
__device__ inline uint32_t backwards(uint32_t block, uint32_t blocks) {
    const uint32_t whole = blocks & ~7u;
    return block < whole ? whole - 8 - (block & ~7u) + (block & 7u) : block;
}

// ---------------------------------------------------------------------------- [n][c][hw]: L lanes to a row
// A group of L lanes takes one channel and BOARDS_AT_ONCE boards: that many loads in flight, the channel's numbers loaded
// once, and the boards' sums joined in registers before they leave (a chunk).  The groups of a workgroup lie along the
// channels, so what it loads at once is one stretch of memory; where there are fewer channels than groups, `abreast`
// boards lie side by side.
//
// How a row fits its lanes (a row of up to 64 pieces of 16 bytes takes one piece a lane, all boards' loads issued before
// the first is used):
//   EXACT  hw is L pieces.
//   ONE    up to L pieces, the last one moved back to end with the row: no partial loads or stores.  The values that it
//          shares with its neighbour are left out of the sums and stored twice, the same.
//   LOOP   longer rows, and rows shorter than a piece: round after round, the last piece value by value.
constexpr int BOARDS_AT_ONCE = 4;
enum Fit { EXACT, ONE, LOOP };

struct RowGrid {
    uint32_t wide, abreast, across;          // channels and boards side by side in a workgroup; workgroups to a board
    uint32_t blocks;
};

static RowGrid row_grid(const NormParams& p, int lanes) {
    const uint32_t groups = NORM_THREADS / lanes, c = (uint32_t)p.c;
    RowGrid g;
    g.wide = c < groups ? c : groups;
    g.abreast = groups / g.wide;
    g.across = (c + groups - 1) / groups;
    g.blocks = (uint32_t)((p.n + BOARDS_AT_ONCE * g.abreast - 1) / (BOARDS_AT_ONCE * g.abreast)) * g.across;
    return g;
}

template <typename T, int L, Fit FIT>
struct RowPlace {
    static constexpr int V = Pack<T>::V;
    uint32_t c, chunk, lane, abreast;
    int64_t n_first;                         // first board; the others follow `abreast` apart
    bool on;
    int off, own;                            // EXACT, ONE: where the lane's piece begins, and its first value that is its own

    __device__ RowPlace(const NormParams& p, const RowGrid& g, uint32_t block) {
        const uint32_t group = threadIdx.x / L, nb = block / g.across, beside = g.abreast == 1 ? 0 : group / g.wide;
        lane = threadIdx.x % L;
        c = block % g.across * (NORM_THREADS / L) + group - beside * g.wide;
        chunk = nb * g.abreast + beside;
        abreast = g.abreast;
        n_first = (int64_t)nb * BOARDS_AT_ONCE * g.abreast + beside;
        on = c < (uint32_t)p.c && beside < g.abreast;
        const int at = lane * V;
        off = FIT == EXACT || at < p.hw - V ? at : p.hw - V;
        own = FIT == EXACT ? 0 : at - off < V ? at - off : V;
    }
    __device__ int64_t board(int k) const { return n_first + k * abreast; }
    __device__ size_t row(const NormParams& p, int k) const { return (size_t)(board(k) < p.n ? board(k) : n_first) * p.c + c; }
    __device__ bool has_piece(const NormParams& p) const { return FIT == EXACT || (int)lane < p.nvec; }
};

// FULL: the piece is whole.
template <bool FULL, typename T>
__device__ inline typename Pack<T>::f32 load_piece(const T* p, int left) { return load_pack(p, FULL ? Pack<T>::V : left); }
template <bool FULL, typename T>
__device__ inline void store_piece(T* p, typename Pack<T>::f32 v, int left) { store_pack(p, v, FULL ? Pack<T>::V : left); }

// f(piece, values left in the row, whether it is whole) for the lane's pieces of a long row: the whole ones four at a time,
// their loads under way together, then the rest of the row.
template <int L, int V, typename F>
__device__ inline void over_pieces(const NormParams& p, int lane, F&& f) {
    const int whole = p.hw / V;
#pragma unroll 4
    for (int j = lane; j < whole; j += L) f(j, V, std::true_type());
    if (whole < p.nvec && lane == whole % L) f(whole, p.hw - whole * V, std::false_type());
}

template <typename T> __device__ inline typename Pack<T>::raw load_raw(const T* p) { return *(const typename Pack<T>::loose*)p; }
template <typename T> __device__ inline typename Pack<T>::f32 widen(typename Pack<T>::raw v) { return __builtin_convertvector(v, typename Pack<T>::f32); }
template <typename T> __device__ inline void store_raw(T* p, typename Pack<T>::f32 v) {
    *(typename Pack<T>::loose*)p = __builtin_convertvector(v, typename Pack<T>::raw);
}

// Mean and centred sum of some values, to which others' are joined: all terms are squares, so nothing cancels whatever the
// values' order.  (The reciprocal is approximate: a mean that is off by d adds count d^2 only.)
struct Centred {
    float mean = 0.f, m2 = 0.f, count = 0.f;
    __device__ void join(float other, float other_m2, float others) {
        const float d = other - mean, before = count;
        count += others;
        const float share = others * __builtin_amdgcn_rcpf(count);
        mean += d * share;
        m2 += other_m2 + d * d * before * share;
    }
};

// Mean and centred sum of a board's values, joined to a chunk's.
struct ChunkStats {
    float mean = 0.f, m2 = 0.f, boards = 0.f;
    __device__ void join(float board, float board_m2, float hw) {
        boards += 1.f;
        const float d = board - mean;
        mean += d / boards;
        m2 += board_m2 + hw * d * (board - mean);
    }
};

template <typename T, int L, Fit FIT, bool GATED>
__global__ __launch_bounds__(NORM_THREADS) void k_row_stats(const T* __restrict__ x, const NormParams p, const RowGrid grid) {
    constexpr int V = Pack<T>::V;
    const RowPlace<T, L, FIT> r(p, grid, blockIdx.x);
    if (!r.on) return;                       // whole groups: the sums below stay within one
    const float hw = (float)p.hw;
    ChunkStats chunk;
    if (r.n_first < p.n) {
        if constexpr (FIT != LOOP) {
            typename Pack<T>::raw raw[BOARDS_AT_ONCE];
#pragma unroll
            for (int k = 0; k < BOARDS_AT_ONCE; ++k) raw[k] = load_raw(x + r.row(p, k) * p.hw + r.off);
#pragma unroll
            for (int k = 0; k < BOARDS_AT_ONCE; ++k) {
                const auto v = widen<T>(raw[k]);
                float s = 0.f, ss = 0.f;
#pragma unroll
                for (int i = 0; i < V; ++i) s += FIT == EXACT || i >= r.own ? v[i] : 0.f;
                const float mean = lane_sum<L>(s) / hw;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float d = FIT == EXACT || i >= r.own ? v[i] - mean : 0.f;
                    ss += d * d;
                }
                ss = lane_sum<L>(ss);
                if (r.board(k) >= p.n) continue;
                if (GATED && r.lane == 0) p.board_mean[r.row(p, k)] = mean;
                chunk.join(mean, ss, hw);
            }
        } else {
            for (int k = 0; k < BOARDS_AT_ONCE && r.board(k) < p.n; ++k) {
                const T* xr = x + r.row(p, k) * p.hw;
                const float first = (float)xr[0];
                Centred own;                 // of the lane's values less the row's first
                over_pieces<L, V>(p, r.lane, [&](int j, int left, auto whole) {
                    const auto v = load_piece<decltype(whole)::value>(xr + j * V, left);
                    const float count = (float)(left < V ? left : V);
                    float s = 0.f, ss = 0.f;
#pragma unroll
                    for (int i = 0; i < V; ++i) s += i < left ? v[i] - first : 0.f;
                    const float mean = s / count;
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float d = i < left ? v[i] - first - mean : 0.f;
                        ss += d * d;
                    }
                    own.join(mean, ss, count);
                });
                const float about = lane_sum<L>(own.count * own.mean) / hw, d = own.mean - about;
                const float ss = lane_sum<L>(own.m2 + own.count * d * d), mean = first + about;
                if (GATED && r.lane == 0) p.board_mean[r.row(p, k)] = mean;
                chunk.join(mean, ss, hw);
            }
        }
    }
    if (r.lane == 0) {
        p.part_a[(size_t)r.chunk * p.c + r.c] = chunk.mean;
        p.part_b[(size_t)r.chunk * p.c + r.c] = chunk.m2;
    }
}

// relu of v, and where it lets the gradient through: where the value is positive, or a NaN (as torch's does)
template <typename F>
__device__ inline uint32_t relu_bits(F& v) {
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(F) / 4); ++i) {
        bits |= (v[i] <= 0.f ? 0u : 1u) << i;
        v[i] = not_below_zero(v[i]);
    }
    return bits;
}

template <typename T, int L, Fit FIT, bool GATED>
__global__ __launch_bounds__(NORM_THREADS) void k_row_apply(const T* __restrict__ x, const T* __restrict__ residual,
                                                            T* __restrict__ out, const NormParams p, const RowGrid grid) {
    constexpr int V = Pack<T>::V;
    const RowPlace<T, L, FIT> r(p, grid, backwards(blockIdx.x, grid.blocks));
    if (!r.on || r.n_first >= p.n) return;
    if constexpr (FIT != LOOP) {
        typename Pack<T>::raw raw[BOARDS_AT_ONCE], res[BOARDS_AT_ONCE];
        float A[BOARDS_AT_ONCE], B[BOARDS_AT_ONCE];
        const float mean = p.mean[r.c];
#pragma unroll
        for (int k = 0; k < BOARDS_AT_ONCE; ++k) {
            const size_t row = r.row(p, k);
            A[k] = p.A[GATED ? row : r.c];
            B[k] = p.B[GATED ? row : r.c];
            raw[k] = load_raw(x + row * p.hw + r.off);
            if (GATED) res[k] = load_raw(residual + row * p.hw + r.off);
        }
#pragma unroll
        for (int k = 0; k < BOARDS_AT_ONCE; ++k) {
            if (r.board(k) >= p.n) return;
            const size_t row = r.row(p, k);
            auto v = (widen<T>(raw[k]) - mean) * A[k] + B[k];
            if (GATED) v += widen<T>(res[k]);
            const uint32_t bits = relu_bits(v);
            store_raw(out + row * p.hw + r.off, v);
            if (r.has_piece(p)) p.mask[row * p.nvec + r.lane] = (uint8_t)bits;
        }
    } else {
        for (int k = 0; k < BOARDS_AT_ONCE && r.board(k) < p.n; ++k) {
            const size_t row = r.row(p, k), at = row * p.hw;
            const float A = p.A[GATED ? row : r.c], B = p.B[GATED ? row : r.c], mean = p.mean[r.c];
            over_pieces<L, V>(p, r.lane, [&](int j, int left, auto whole) {
                constexpr bool FULL = decltype(whole)::value;
                auto v = (load_piece<FULL>(x + at + j * V, left) - mean) * A + B;
                if (GATED) v += load_piece<FULL>(residual + at + j * V, left);
                const uint32_t bits = relu_bits(v);
                store_piece<FULL>(out + at + j * V, v, left);
                p.mask[row * p.nvec + j] = (uint8_t)bits;
            });
        }
    }
}

template <typename T, int L, Fit FIT, bool GATED>
__global__ __launch_bounds__(NORM_THREADS) void k_row_grad_sums(const T* __restrict__ x, const T* __restrict__ grad,
                                                                T* __restrict__ dresidual, const NormParams p, const RowGrid grid) {
    constexpr int V = Pack<T>::V;
    const RowPlace<T, L, FIT> r(p, grid, blockIdx.x);
    if (!r.on) return;
    const float mean = p.mean[r.c];
    float a = 0.f, b = 0.f;
    const auto board_sums = [&](int k, float s1, float s2) {
        if (GATED) {                         // the gate's gradient needs every board's
            s1 = lane_sum<L>(s1);
            s2 = lane_sum<L>(s2);
            if (r.board(k) < p.n && r.lane == 0) {
                p.s1[r.row(p, k)] = s1;
                p.s2[r.row(p, k)] = s2;
            }
        } else if (r.board(k) < p.n) {
            a += s1;
            b += s2;
        }
    };
    if (r.n_first < p.n) {
        if constexpr (FIT != LOOP) {
            typename Pack<T>::raw raw[BOARDS_AT_ONCE], gr[BOARDS_AT_ONCE];
            uint32_t bits[BOARDS_AT_ONCE];
            const uint32_t piece = r.has_piece(p) ? r.lane : 0;
#pragma unroll
            for (int k = 0; k < BOARDS_AT_ONCE; ++k) {
                const size_t row = r.row(p, k);
                raw[k] = load_raw(x + row * p.hw + r.off);
                gr[k] = load_raw(grad + row * p.hw + r.off);
                bits[k] = p.mask[row * p.nvec + piece];
            }
#pragma unroll
            for (int k = 0; k < BOARDS_AT_ONCE; ++k) {
                const auto v = widen<T>(raw[k]);
                auto g = widen<T>(gr[k]);
                float s1 = 0.f, s2 = 0.f;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    g[i] = bits[k] >> i & 1 ? g[i] : 0.f;
                    const float gi = FIT == EXACT || i >= r.own ? g[i] : 0.f;
                    s1 += gi;
                    s2 += gi * (v[i] - mean);
                }
                if (GATED && r.board(k) < p.n && r.has_piece(p)) store_raw(dresidual + r.row(p, k) * p.hw + r.off, g);
                board_sums(k, s1, s2);
            }
        } else {
            for (int k = 0; k < BOARDS_AT_ONCE && r.board(k) < p.n; ++k) {
                const size_t row = r.row(p, k), at = row * p.hw;
                float s1 = 0.f, s2 = 0.f;
                over_pieces<L, V>(p, r.lane, [&](int j, int left, auto whole) {
                    constexpr bool FULL = decltype(whole)::value;
                    const auto v = load_piece<FULL>(x + at + j * V, left);
                    auto g = load_piece<FULL>(grad + at + j * V, left);
                    const uint32_t bits = p.mask[row * p.nvec + j];
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        g[i] = bits >> i & 1 ? g[i] : 0.f;
                        s1 += g[i];
                        s2 += g[i] * (v[i] - mean);
                    }
                    if (GATED) store_piece<FULL>(dresidual + at + j * V, g, left);
                });
                board_sums(k, s1, s2);
            }
        }
    }
    if (!GATED) {
        a = lane_sum<L>(a);
        b = lane_sum<L>(b);
        if (r.lane == 0) {
            p.part_a[(size_t)r.chunk * p.c + r.c] = a;
            p.part_b[(size_t)r.chunk * p.c + r.c] = b;
        }
    }
}

// grad: the masked one (dresidual) if gated
template <typename T, int L, Fit FIT, bool GATED>
__global__ __launch_bounds__(NORM_THREADS) void k_row_grad_apply(const T* __restrict__ x, const T* __restrict__ grad,
                                                                 T* __restrict__ dx, const NormParams p, const RowGrid grid, uint32_t joins) {
    constexpr int V = Pack<T>::V;
    if (GATED && blockIdx.x < joins) {
        join_weights(p, blockIdx.x);
        return;
    }
    const RowPlace<T, L, FIT> r(p, grid, backwards(blockIdx.x - joins, grid.blocks));
    if (!r.on || r.n_first >= p.n) return;
    const float mean = p.mean[r.c], inv = p.inv[r.c], b = p.cb[r.c], ca = p.ca[r.c], cd = p.cd[r.c], per_place = ca / (float)p.hw;
    if constexpr (FIT != LOOP) {
        typename Pack<T>::raw raw[BOARDS_AT_ONCE], gr[BOARDS_AT_ONCE];
        float gate[BOARDS_AT_ONCE], dq[BOARDS_AT_ONCE];
        uint32_t bits[BOARDS_AT_ONCE];
        const uint32_t piece = r.has_piece(p) ? r.lane : 0;
#pragma unroll
        for (int k = 0; k < BOARDS_AT_ONCE; ++k) {
            const size_t row = r.row(p, k);
            if (GATED) {
                gate[k] = p.gate[row];
                dq[k] = p.dq[row];
            } else {
                bits[k] = p.mask[row * p.nvec + piece];
            }
            raw[k] = load_raw(x + row * p.hw + r.off);
            gr[k] = load_raw(grad + row * p.hw + r.off);
        }
#pragma unroll
        for (int k = 0; k < BOARDS_AT_ONCE; ++k) {
            if (r.board(k) >= p.n) return;
            const float a = GATED ? ca * gate[k] : ca, d = GATED ? cd + per_place * dq[k] : cd;
            const auto v = widen<T>(raw[k]);
            auto g = widen<T>(gr[k]);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (!GATED) g[i] = bits[k] >> i & 1 ? g[i] : 0.f;
                g[i] = g[i] * a + (p.training ? (v[i] - mean) * inv * b + d : d);
            }
            if (r.has_piece(p)) store_raw(dx + r.row(p, k) * p.hw + r.off, g);
        }
    } else {
        for (int k = 0; k < BOARDS_AT_ONCE && r.board(k) < p.n; ++k) {
            const size_t row = r.row(p, k), at = row * p.hw;
            const float a = GATED ? ca * p.gate[row] : ca, d = GATED ? cd + per_place * p.dq[row] : cd;
            over_pieces<L, V>(p, r.lane, [&](int j, int left, auto whole) {
                constexpr bool FULL = decltype(whole)::value;
                const auto v = load_piece<FULL>(x + at + j * V, left);
                auto g = load_piece<FULL>(grad + at + j * V, left);
                const uint32_t bits = GATED ? 0 : p.mask[row * p.nvec + j];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    if (!GATED) g[i] = bits >> i & 1 ? g[i] : 0.f;
                    g[i] = g[i] * a + (p.training ? (v[i] - mean) * inv * b + d : d);
                }
                store_piece<FULL>(dx + at + j * V, g, left);
            });
        }
    }
}

// ---------------------------------------------- [n][hw][c]: a workgroup to a board and a range of channels
// Thread (ty, tx): 16 bytes of channels, every ty-th place of the board; the ty are added through LDS.  A chunk is a board.
// The last 16 bytes are moved back to end with the channels (what they share with their neighbours is computed twice, the
// same); fewer channels than 16 bytes go value by value.
struct Lanes {
    int tx, ty, step;          // step: places taken at once
    int j;                     // which 16 bytes of the channels
    bool on;
    int c, left;               // first channel, channels from there on
};

template <typename T>
__device__ inline Lanes lanes_of(const NormParams& p, int wide) {
    constexpr int V = Pack<T>::V;
    Lanes l;
    l.tx = threadIdx.x % wide;
    l.ty = threadIdx.x / wide;
    l.step = NORM_THREADS / wide;
    l.j = blockIdx.y * wide + l.tx;
    l.on = l.ty < l.step && l.j < p.nvec;
    l.c = p.c >= V && l.j * V > p.c - V ? p.c - V : l.j * V;
    l.left = p.c - l.c;
    return l;
}

// Numbers of the thread's channels, 16 bytes at a time.
template <typename F>
__device__ inline F load_channels(const float* p, int left) {
    constexpr int V = sizeof(F) / 4;
    F r;
#pragma unroll
    for (int i = 0; i < V; i += 4) {
        const f32x4 v = load_pack(p + i, left - i);
#pragma unroll
        for (int k = 0; k < 4; ++k) r[i + k] = v[k];
    }
    return r;
}

// The threads' values of one channel through the LDS; out(c, a, b, stride) for each of the workgroup's channels: thread ty's
// are a[ty * stride] and b[ty * stride].
template <int V, typename F, typename Out>
__device__ inline void over_places(F a, F b, const Lanes& l, const NormParams& p, int wide, Out&& out) {
    __shared__ float red[2][NORM_THREADS * V];
    if (l.ty < l.step) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            red[0][(l.ty * wide + l.tx) * V + i] = a[i];
            red[1][(l.ty * wide + l.tx) * V + i] = b[i];
        }
    }
    __syncthreads();
    const int c0 = blockIdx.y * wide * V;
    for (int i = threadIdx.x; i < wide * V; i += NORM_THREADS) {
        // channel of the i-th value: the last piece is moved back
        const int piece = c0 + i / V * V, c = (p.c >= V && piece > p.c - V && piece < p.c ? p.c - V : piece) + i % V;
        if (c < p.c) out(c, red[0] + i, red[1] + i, wide * V);
    }
}

// Sums over the places; out(c, a, b) for each of the workgroup's channels.
template <int V, typename F, typename Out>
__device__ inline void add_places(F a, F b, const Lanes& l, const NormParams& p, int wide, Out&& out) {
    over_places<V>(a, b, l, p, wide, [&](int c, const float* u, const float* v, int stride) {
        float s = 0.f, ss = 0.f;
        for (int y = 0; y < l.step; ++y) {
            s += u[y * stride];
            ss += v[y * stride];
        }
        out(c, s, ss);
    });
}

template <typename T, bool FULL, bool GATED>
__global__ __launch_bounds__(NORM_THREADS) void k_last_stats(const T* __restrict__ x, const NormParams p, int wide) {
    constexpr int V = Pack<T>::V;
    typedef typename Pack<T>::f32 F;
    const Lanes l = lanes_of<T>(p, wide);
    const T* xb = x + (size_t)blockIdx.x * p.hw * p.c;
    F mean, m2;                              // of the thread's values less the board's first (one by one as in Centred)
#pragma unroll
    for (int i = 0; i < V; ++i) mean[i] = m2[i] = 0.f;
    if (l.on) {
        const F first = load_piece<FULL>(xb + l.c, l.left);
        float count = 0.f;
#pragma unroll 4
        for (int y = l.ty; y < p.hw; y += l.step) {
            const F v = load_piece<FULL>(xb + (size_t)y * p.c + l.c, l.left) - first, d = v - mean;
            count += 1.f;
            mean += d * __builtin_amdgcn_rcpf(count);
            m2 += d * (v - mean);
        }
    }
    const float hw = (float)p.hw, each = (float)(p.hw / l.step);
    const int more = p.hw % l.step;          // threads with a place more than the others
    over_places<V>(mean, m2, l, p, wide, [&](int c, const float* means, const float* m2s, int stride) {
        const auto count = [&](int y) { return y < more ? each + 1.f : each; };
        float s = 0.f, ss = 0.f;
#pragma unroll 8
        for (int y = 0; y < l.step; ++y) s += count(y) * means[y * stride];
        const float about = s / hw;
#pragma unroll 8
        for (int y = 0; y < l.step; ++y) {
            const float d = means[y * stride] - about;
            ss += m2s[y * stride] + count(y) * d * d;
        }
        const float mean = (float)xb[c] + about;
        const size_t row = (size_t)blockIdx.x * p.c + c;
        if (GATED) p.board_mean[row] = mean;
        p.part_a[row] = mean;
        p.part_b[row] = ss;
    });
}

template <typename T, bool FULL, bool GATED>
__global__ __launch_bounds__(NORM_THREADS) void k_last_apply(const T* __restrict__ x, const T* __restrict__ residual,
                                                             T* __restrict__ out, const NormParams p, int wide) {
    constexpr int V = Pack<T>::V;
    typedef typename Pack<T>::f32 F;
    const Lanes l = lanes_of<T>(p, wide);
    if (!l.on) return;
    const uint32_t n = backwards(blockIdx.x, gridDim.x);
    const size_t q = (GATED ? (size_t)n * p.c : 0) + l.c;
    const F A = load_channels<F>(p.A + q, l.left), B = load_channels<F>(p.B + q, l.left), mean = load_channels<F>(p.mean + l.c, l.left);
    const size_t board = (size_t)n * p.hw;
#pragma unroll 4
    for (int y = l.ty; y < p.hw; y += l.step) {
        const size_t at = (board + y) * p.c + l.c;
        F v = (load_piece<FULL>(x + at, l.left) - mean) * A + B;
        if (GATED) v += load_piece<FULL>(residual + at, l.left);
        uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            bits |= (v[i] <= 0.f ? 0u : 1u) << i;
            v[i] = not_below_zero(v[i]);
        }
        store_piece<FULL>(out + at, v, l.left);
        p.mask[(board + y) * p.nvec + l.j] = (uint8_t)bits;
    }
}

template <typename T, bool FULL, bool GATED>
__global__ __launch_bounds__(NORM_THREADS) void k_last_grad_sums(const T* __restrict__ x, const T* __restrict__ grad,
                                                                 T* __restrict__ dresidual, const NormParams p, int wide) {
    constexpr int V = Pack<T>::V;
    typedef typename Pack<T>::f32 F;
    const Lanes l = lanes_of<T>(p, wide);
    F s1, s2;
#pragma unroll
    for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.f;
    const size_t board = (size_t)blockIdx.x * p.hw;
    if (l.on) {
        const F mean = load_channels<F>(p.mean + l.c, l.left);
#pragma unroll 4
        for (int y = l.ty; y < p.hw; y += l.step) {
            const size_t at = (board + y) * p.c + l.c;
            const F v = load_piece<FULL>(x + at, l.left);
            F g = load_piece<FULL>(grad + at, l.left);
            const uint32_t bits = p.mask[(board + y) * p.nvec + l.j];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                g[i] = bits >> i & 1 ? g[i] : 0.f;
                s1[i] += g[i];
                s2[i] += g[i] * (v[i] - mean[i]);
            }
            if (GATED) store_piece<FULL>(dresidual + at, g, l.left);
        }
    }
    float *a = GATED ? p.s1 : p.part_a, *b = GATED ? p.s2 : p.part_b;
    add_places<V>(s1, s2, l, p, wide, [&](int c, float u, float v) {
        a[(size_t)blockIdx.x * p.c + c] = u;
        b[(size_t)blockIdx.x * p.c + c] = v;
    });
}

template <typename T, bool FULL, bool GATED>
__global__ __launch_bounds__(NORM_THREADS) void k_last_grad_apply(const T* __restrict__ x, const T* __restrict__ grad,
                                                                  T* __restrict__ dx, const NormParams p, int wide, uint32_t joins) {
    constexpr int V = Pack<T>::V;
    typedef typename Pack<T>::f32 F;
    if (GATED && blockIdx.x < joins) {
        if (blockIdx.y == 0) join_weights(p, blockIdx.x);
        return;
    }
    const uint32_t n = backwards(blockIdx.x - joins, gridDim.x - joins);
    const Lanes l = lanes_of<T>(p, wide);
    if (!l.on) return;
    const size_t row = (size_t)n * p.c + l.c;
    const F mean = load_channels<F>(p.mean + l.c, l.left), inv = load_channels<F>(p.inv + l.c, l.left), b = load_channels<F>(p.cb + l.c, l.left);
    F a = load_channels<F>(p.ca + l.c, l.left), d = load_channels<F>(p.cd + l.c, l.left);
    if (GATED) {
        d += a * load_channels<F>(p.dq + row, l.left) / (float)p.hw;
        a *= load_channels<F>(p.gate + row, l.left);
    }
    const size_t board = (size_t)n * p.hw;
#pragma unroll 4
    for (int y = l.ty; y < p.hw; y += l.step) {
        const size_t at = (board + y) * p.c + l.c;
        const F v = load_piece<FULL>(x + at, l.left);
        F g = load_piece<FULL>(grad + at, l.left);
        const uint32_t bits = GATED ? 0 : p.mask[(board + y) * p.nvec + l.j];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (!GATED) g[i] = bits >> i & 1 ? g[i] : 0.f;
            g[i] = g[i] * a[i] + (p.training ? (v[i] - mean[i]) * inv[i] * b[i] + d[i] : d[i]);
        }
        store_piece<FULL>(dx + at, g, l.left);
    }
}

// ------------------------------------------------------------ per channel: sums over chunks of boards in 64 bits
constexpr int CHANNELS = 8, LINES = 64;       // a workgroup: 8 neighbouring channels, 64 chunks at a time
constexpr int IN_FLIGHT = 8;                  // chunks whose loads a thread has under way

// Sums of v over the threads of a channel; thread 0 to CHANNELS - 1 get theirs.
template <int K>
__device__ inline void add_lines(double (&v)[K]) {
    __shared__ double red[CHANNELS * LINES / 64][CHANNELS][K];
#pragma unroll
    for (int k = 0; k < K; ++k)
        for (int off = CHANNELS; off < 64; off <<= 1) v[k] += __shfl_xor(v[k], off);
    const int lane = threadIdx.x & 63;
    if (lane < CHANNELS)
#pragma unroll
        for (int k = 0; k < K; ++k) red[threadIdx.x >> 6][lane][k] = v[k];
    __syncthreads();
    if (threadIdx.x < CHANNELS)
#pragma unroll
        for (int k = 0; k < K; ++k)
            for (int w = 1; w < CHANNELS * LINES / 64; ++w) v[k] += red[w][threadIdx.x][k];
}

// term(i, a, b) for every chunk i of the thread's channel c.
template <typename F>
__device__ inline void over_chunks(const NormParams& p, int c, F&& term) {
    if (c >= p.c) return;
    for (int64_t i = threadIdx.x / CHANNELS; i < p.chunks; i += LINES * IN_FLIGHT) {
        float a[IN_FLIGHT], b[IN_FLIGHT];
#pragma unroll
        for (int u = 0; u < IN_FLIGHT; ++u) {
            const int64_t iu = i + u * LINES, at = (iu < p.chunks ? iu : i) * p.c + c;
            a[u] = p.part_a[at];
            b[u] = p.part_b[at];
        }
#pragma unroll
        for (int u = 0; u < IN_FLIGHT; ++u)
            if (i + u * LINES < p.chunks) term(i + u * LINES, a[u], b[u]);
    }
}

__global__ __launch_bounds__(CHANNELS * LINES) void k_channel_stats(const NormParams p) {
    const int c = blockIdx.x * CHANNELS + threadIdx.x % CHANNELS;
    const bool mine = threadIdx.x < CHANNELS && c < p.c;
    float old_mean = 0.f, old_var = 0.f, weight = 0.f, bias = 0.f;
    if (mine) {                       // under way during the sums
        if (p.running_mean) old_mean = p.running_mean[c];
        if (p.running_var) old_var = p.running_var[c];
        weight = p.weight[c];
        bias = p.bias[c];
    }
    double v[3] = {0, 0, 0};          // sums over the boards: of their means, of the means' squares, of the centred sums
    if (p.training) {
        over_chunks(p, c, [&](int64_t i, float mean, float m2) {
            const double k = boards_in_chunk(p, (uint32_t)i), m = mean;
            v[0] += k * m;
            v[1] += k * (m * m);
            v[2] += m2;
        });
        add_lines(v);
    }
    if (mine) {
        double mean, var;
        if (p.training) {
            const double count = (double)p.n * p.hw;
            mean = v[0] / p.n;
            var = (v[2] + p.hw * (v[1] - p.n * mean * mean)) / count;
            if (var < 0.0) var = 0.0;          // a NaN stays one
            if (p.running_mean) p.running_mean[c] = (float)((1.0 - p.momentum) * old_mean + p.momentum * mean);
            if (p.running_var) p.running_var[c] = (float)((1.0 - p.momentum) * old_var + p.momentum * var * count / (count - 1.0));
        } else {
            mean = old_mean;
            var = old_var;
        }
        const float inv = (float)(1.0 / sqrt(var + p.eps)), m = (float)mean;
        p.mean[c] = m;
        p.inv[c] = inv;
        if (!p.hidden) {
            p.A[c] = weight * inv;
            p.B[c] = bias;
        }
    }
    if (p.num_batches && p.training && blockIdx.x == 0 && threadIdx.x == 0) *p.num_batches += 1;
}

// dy's channel sums, and with them what the last pass needs: dx = ca gm (gate) + xc / s cb + cd (+ ca dq / hw), without
// cb and cd where the statistics are the running ones (not with zeros: x may be infinite)
__device__ inline void channel_grads(const NormParams& p, int block) {
    const int c = block * CHANNELS + threadIdx.x % CHANNELS;
    const bool mine = threadIdx.x < CHANNELS && c < p.c;
    const float inv = mine ? p.inv[c] : 0.f, a = mine ? p.weight[c] * inv : 0.f;
    double v[2] = {0, 0};
    over_chunks(p, c, [&](int64_t, float s1, float s2) {
        v[0] += s1;
        v[1] += s2;
    });
    add_lines(v);
    if (mine) {
        const double count = (double)p.n * p.hw;
        p.dbias[c] = (float)v[0];
        p.dweight[c] = (float)(v[1] * inv);
        p.ca[c] = a;
        p.cb[c] = p.training ? (float)(-a * (v[1] * inv / count)) : 0.f;
        p.cd[c] = p.training ? (float)(-a * (v[0] / count)) : 0.f;
    }
}

// --------------------------------------------------------------------------------------------- the gate
// A workgroup takes four boards: their vectors lie in the LDS as [element][board], so one 16-byte read serves four boards
// and a weight is loaded once for all of them.  Weights are read along their rows, 16 bytes a lane.  Four dependent
// round trips to memory bound it (statistics, fc1, fc2, results): 6.4 us forward and 6.8 us backward at 1024 boards of 128
// channels and 16 hidden units, 17 us each at 4096 x 256 x 32.  (There, eight boards to a workgroup: 20 and 21 us, half the
// weights' traffic but half the workgroups to wait for it; eight rows ahead: 21 and 17.)
constexpr int GATE_THREADS = 256;

// Four weights from p on; FOURS: the rows are multiples of four.
template <bool FOURS>
__device__ inline f32x4 four_weights(const float* p, int left) {
    return FOURS ? *(const f32x4_loose*)p : load_pack(p, left);
}

template <typename F>
__device__ inline void with_fours(int cols, F&& f) {
    if (cols % 4 == 0) f(std::true_type());
    else f(std::false_type());
}

// out(j, bias[j] + row j of w [rows][cols] against the four boards' vectors v).  L lanes to a row, ROWS_AHEAD rows' loads
// under way; every lane of them gets the sums.
constexpr int ROWS_AHEAD = 4;

template <int L, bool FOURS, typename F>
__device__ inline void rows_times(const float* w, const float* bias, int rows, int cols, const f32x4* v, F&& out) {
    constexpr int STEP = GATE_THREADS / L;
    const int lane = threadIdx.x % L;
    for (int j0 = threadIdx.x / L; j0 < rows; j0 += STEP * ROWS_AHEAD) {
        f32x4 s[ROWS_AHEAD];
#pragma unroll
        for (int u = 0; u < ROWS_AHEAD; ++u) s[u] = lane == 0 ? bias[j0 + u * STEP < rows ? j0 + u * STEP : j0] : 0.f;
        for (int c = lane * 4; c < cols; c += L * 4) {
            f32x4 q[ROWS_AHEAD];
#pragma unroll
            for (int u = 0; u < ROWS_AHEAD; ++u) {
                const int j = j0 + u * STEP;
                q[u] = four_weights<FOURS>(w + (size_t)(j < rows ? j : j0) * cols + c, cols - c);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 vi = v[FOURS || c + i < cols ? c + i : 0];
#pragma unroll
                for (int u = 0; u < ROWS_AHEAD; ++u) s[u] += q[u][i] * vi;
            }
        }
#pragma unroll
        for (int u = 0; u < ROWS_AHEAD; ++u) {
#pragma unroll
            for (int r = 0; r < 4; ++r) s[u][r] = lane_sum<L>(s[u][r]);
            const int j = j0 + u * STEP;
            if (j < rows) out(j, s[u]);
        }
    }
}

template <typename F>
__device__ inline void rows_times(const float* w, const float* bias, int rows, int cols, const f32x4* v, F&& out) {
    with_fours(cols, [&](auto fours) {
        constexpr bool FOURS = decltype(fours)::value;
        if (cols <= 16) rows_times<4, FOURS>(w, bias, rows, cols, v, out);
        else if (cols <= 32) rows_times<8, FOURS>(w, bias, rows, cols, v, out);
        else rows_times<16, FOURS>(w, bias, rows, cols, v, out);
    });
}

// out(k, sums) for every column k: the columns of w against v.  A thread takes four columns and every parts-th row; the parts
// are added through the LDS in `part` (GATE_THREADS * 4 vectors).
template <typename F>
__device__ inline void columns_times(const float* w, int rows, int cols, const f32x4* v, f32x4* part, F&& out) {
    const int fours = (cols + 3) / 4;
    int wide = 1;
    while (wide < fours && wide < GATE_THREADS) wide *= 2;
    const int parts = GATE_THREADS / wide, x = threadIdx.x % wide, y = threadIdx.x / wide;
    for (int at = 0; at < fours; at += wide) {
        const int k = (at + x) * 4;
        f32x4 s[4] = {0.f, 0.f, 0.f, 0.f};
        if (k < cols)
            with_fours(cols, [&](auto whole) {
                // (rows past the end are loaded again and count nothing: a guard on each would make their loads wait in turn)
                for (int j0 = y; j0 < rows; j0 += parts * ROWS_AHEAD) {
                    f32x4 q[ROWS_AHEAD];
#pragma unroll
                    for (int u = 0; u < ROWS_AHEAD; ++u) {
                        const int j = j0 + u * parts;
                        q[u] = four_weights<decltype(whole)::value>(w + (size_t)(j < rows ? j : j0) * cols + k, cols - k);
                    }
#pragma unroll
                    for (int u = 0; u < ROWS_AHEAD; ++u) {
                        const int j = j0 + u * parts;
                        const f32x4 vj = v[j < rows ? j : j0] * (j < rows ? 1.f : 0.f);
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[i] += q[u][i] * vj;
                    }
                }
            });
#pragma unroll
        for (int i = 0; i < 4; ++i) part[(y * wide + x) * 4 + i] = s[i];
        __syncthreads();
        const int share = wide * 4 < GATE_THREADS ? GATE_THREADS / (wide * 4) : 1;                   // lanes to a sum: 1 to 64
        for (int i = threadIdx.x / share; i < wide * 4; i += GATE_THREADS / share) {
            f32x4 t = 0.f;
            for (int q = threadIdx.x % share; q < parts; q += share) t += part[q * wide * 4 + i];
            for (int off = 1; off < share; off <<= 1)
#pragma unroll
                for (int r = 0; r < 4; ++r) t[r] += __shfl_xor(t[r], off);
            if (threadIdx.x % share == 0 && at * 4 + i < cols) out(at * 4 + i, t);
        }
        __syncthreads();
    }
}

__global__ __launch_bounds__(GATE_THREADS) void k_gate_forward(const NormParams p) {
    extern __shared__ f32x4 lds4[];
    f32x4 *q = lds4, *h = q + p.c, *e = h + p.hidden;        // [c], [hidden], [2c]
    const int64_t n0 = (int64_t)blockIdx.x * GATE_ROWS;
    const int rows = (int)(p.n - n0 < GATE_ROWS ? p.n - n0 : GATE_ROWS);
    for (int c = threadIdx.x; c < p.c; c += GATE_THREADS) {
        const float scale = p.weight[c] * p.inv[c], mean = p.mean[c], bias = p.bias[c];
        f32x4 v;
#pragma unroll
        for (int r = 0; r < GATE_ROWS; ++r) v[r] = (p.board_mean[(n0 + (r < rows ? r : 0)) * p.c + c] - mean) * scale + bias;
        q[c] = v;
    }
    __syncthreads();
    rows_times(p.w1, p.b1, p.hidden, p.c, q, [&](int k, f32x4 s) {
#pragma unroll
        for (int r = 0; r < GATE_ROWS; ++r) s[r] = not_below_zero(s[r]);
        h[k] = s;                                            // every lane of the row writes the same
    });
    __syncthreads();
    for (int i = threadIdx.x; i < GATE_ROWS * p.hidden; i += GATE_THREADS) {
        const int r = i / p.hidden, k = i % p.hidden;
        if (r < rows) p.h[(n0 + r) * p.hidden + k] = h[k][r];
    }
    rows_times(p.w2, p.b2, 2 * p.c, p.hidden, h, [&](int j, const f32x4 s) { e[j] = s; });
    __syncthreads();
    for (int c = threadIdx.x; c < p.c; c += GATE_THREADS) {
        const float scale = p.weight[c] * p.inv[c], bias = p.bias[c];
        const f32x4 w = e[c], b = e[p.c + c];
#pragma unroll
        for (int r = 0; r < GATE_ROWS; ++r)
            if (r < rows) {
                const int64_t row = (n0 + r) * p.c + c;
                const float gate = 1.f / (1.f + expf(-w[r]));
                p.gate[row] = gate;
                p.A[row] = scale * gate;
                p.B[row] = bias * gate + b[r];
            }
    }
}

__global__ __launch_bounds__(GATE_THREADS) void k_gate_backward(const NormParams p) {
    extern __shared__ f32x4 lds4[];
    f32x4 *de = lds4, *dh = de + 2 * p.c, *part = dh + p.hidden;     // [2c], [hidden], [GATE_THREADS * 4]
    const int64_t n0 = (int64_t)blockIdx.x * GATE_ROWS;
    const int rows = (int)(p.n - n0 < GATE_ROWS ? p.n - n0 : GATE_ROWS);
    // (a board past the end is read as the first one and not written: a guard on each load would make them wait in turn)
    const auto board = [&](int r) { return n0 + (r < rows ? r : 0); };
    for (int c = threadIdx.x; c < p.c; c += GATE_THREADS) {
        const float scale = p.weight[c] * p.inv[c], bias = p.bias[c];
        f32x4 gate, s1, s2;
#pragma unroll
        for (int r = 0; r < GATE_ROWS; ++r) {
            const int64_t row = board(r) * p.c + c;
            gate[r] = p.gate[row];
            s1[r] = p.s1[row];
            s2[r] = p.s2[row];
        }
        const f32x4 w = gate * (1.f - gate) * (scale * s2 + bias * s1);
        de[c] = w;
        de[p.c + c] = s1;
#pragma unroll
        for (int r = 0; r < GATE_ROWS; ++r)
            if (r < rows) {
                p.de[(n0 + r) * 2 * p.c + c] = w[r];
                p.de[(n0 + r) * 2 * p.c + p.c + c] = s1[r];
            }
    }
    __syncthreads();
    columns_times(p.w2, 2 * p.c, p.hidden, de, part, [&](int k, f32x4 s) {
        f32x4 h;
#pragma unroll
        for (int r = 0; r < GATE_ROWS; ++r) h[r] = p.h[board(r) * p.hidden + k];
#pragma unroll
        for (int r = 0; r < GATE_ROWS; ++r) {
            if (h[r] <= 0.f) s[r] = 0.f;
            if (r < rows) p.dh[(n0 + r) * p.hidden + k] = s[r];
        }
        dh[k] = s;
    });
    columns_times(p.w1, p.hidden, p.c, dh, part, [&](int c, const f32x4 s) {
        // this workgroup's share of dy's channel sums
        const float mean = p.mean[c];
        f32x4 gate, s1, s2, m;
#pragma unroll
        for (int r = 0; r < GATE_ROWS; ++r) {
            const int64_t row = board(r) * p.c + c;
            gate[r] = p.gate[row];
            s1[r] = p.s1[row];
            s2[r] = p.s2[row];
            m[r] = p.board_mean[row];
        }
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int r = 0; r < GATE_ROWS; ++r)
            if (r < rows) {
                p.dq[(n0 + r) * p.c + c] = s[r];
                a += gate[r] * s1[r] + s[r];
                b += gate[r] * s2[r] + s[r] * (m[r] - mean);
            }
        p.part_a[(size_t)blockIdx.x * p.c + c] = a;
        p.part_b[(size_t)blockIdx.x * p.c + c] = b;
    });
}

// Gradients of the gate's weights: sums over the boards of outer products, as 32 x 32 tiles on the matrix unit (in
// float32: two boards an instruction, a lane loads one value of each factor).  A workgroup takes one tile and one of
// `splits` ranges of boards, its wavefronts two boards in turn, the loads of 16 boards in flight.  The bias is the sum of
// the left factor.  The partial tiles go to the workspace; the last pass's first workgroups add them in order, beside
// its own work.
constexpr int TILE = 32, TILE_WAVES = CHANNELS * LINES / 64, TILE_AHEAD = 8, TILE_OUT = TILE * TILE + TILE;

struct TileShape {
    int m, k, across, tiles;                                         // [m][k] in `tiles` tiles, `across` to a row
};

__host__ __device__ inline TileShape tile_shape(int m, int k) {
    const int across = (k + TILE - 1) / TILE;
    return {m, k, across, (m + TILE - 1) / TILE * across};
}

__host__ __device__ inline int weight_tiles(const NormParams& p) { return tile_shape(2 * p.c, p.hidden).tiles + tile_shape(p.hidden, p.c).tiles; }

// Ranges of at least 64 boards, and no more workgroups than twice the compute units: every range is a partial tile more
// to join.  (At 4096 x 256, 24 tiles: 21 ranges 12.9 us, 10 ranges 16.7; 64 ranges would cost the pass that joins them
// 7 us more.  At 1024 x 128, 12 tiles: 16 ranges 4.7 us, 8 ranges 5.1.)
__host__ __device__ inline int weight_splits(const NormParams& p) {
    const int64_t most = (p.n + 63) / 64, enough = 512 / weight_tiles(p);
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
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, at = lane & 31, second_board = lane >> 5;
    // (a lane past the end of a factor reads its last value; what comes of it is not joined)
    const int i = i0 + at < t.m ? i0 + at : t.m - 1, j = j0 + at < t.k ? j0 + at : t.k - 1;
    const float *left = (second ? p.de : p.dh) + i, *right = (second ? p.h : p.board_mean) + j;
    // fc1's right factor: q = (mean over the board - mean) * scale + shift
    const float scale = second ? 1.f : p.weight[j] * p.inv[j], shift = second ? 0.f : p.bias[j], mean = second ? 0.f : p.mean[j];
    typedef float f32x16 __attribute__((ext_vector_type(16)));
    f32x16 acc = 0.f;
    float bias = 0.f;
    const int64_t from = p.n * split / splits, to = p.n * (split + 1) / splits;
    for (int64_t n = from + 2 * wave; n < to; n += 2 * TILE_WAVES * TILE_AHEAD) {
        float a[TILE_AHEAD], b[TILE_AHEAD];
#pragma unroll
        for (int u = 0; u < TILE_AHEAD; ++u) {
            const int64_t nu = n + 2 * TILE_WAVES * u + second_board, in = nu < to ? nu : from;
            a[u] = left[in * t.m];
            b[u] = right[in * t.k];
        }
#pragma unroll
        for (int u = 0; u < TILE_AHEAD; ++u) {
            const float w = n + 2 * TILE_WAVES * u + second_board < to ? a[u] : 0.f;
            bias += w;
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(w, (b[u] - mean) * scale + shift, acc, 0, 0, 0);
        }
    }
    bias += __shfl_xor(bias, 32);
#pragma unroll
    for (int r = 0; r < 16; ++r) lds[wave][(8 * (r / 4) + 4 * second_board + r % 4) * TILE + at] = acc[r];
    if (lane < TILE) lds[wave][TILE * TILE + lane] = bias;
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

// (a multiple of eight, so that the workgroups behind them stay on their dies)
static int join_blocks(const NormParams& p) { return p.hidden ? ((weight_tiles(p) * TILE_OUT + NORM_THREADS - 1) / NORM_THREADS + 7) & ~7 : 0; }

__global__ __launch_bounds__(CHANNELS * LINES) void k_param_grads(const NormParams p, int channel_blocks) {
    if ((int)blockIdx.x < channel_blocks) channel_grads(p, blockIdx.x);
    else weight_tile(p, (int)blockIdx.x - channel_blocks);
}

// ------------------------------------------------------------- a plain norm, [n][c][hw]: a workgroup to a channel
// Where a channel's n rows fit a workgroup's registers (8192 pieces of 16 bytes: 1024 boards of 8 x 8 in 16 bits) it is read
// once, its sums are taken there and the result leaves by the same kernel: one launch each way instead of three, 5
// activations instead of 8, and no mask (whether out > 0 follows from x again, by the same operations).  Sums are
// joined in 64 bits; the variance is taken about a first mean, with the remainder's square taken off.
// Neighbouring channels share cache lines, so a die takes a range of them.
// Forward and backward, beside the passes of row sums (all their launches): 37 x 48 x 81 in float16 10 us (22), 128 x 128 x 64 in
// float32 14 (22), 512 x 128 x 64 in float32 24 (31), 8 x 1024 x 361 in float32 16 (39), 1024 x 128 x 64 in bfloat16 30 (34); with
// two channels, so two workgroups, 1024 x 2 x 64 in bfloat16 takes 21 either way.
constexpr int CHANNEL_PIECES = 8192;

__device__ inline uint32_t channel_of(uint32_t block, uint32_t c) {
    const uint32_t die = block % 8, more = c % 8;
    return die * (c / 8) + (die < more ? die : more) + block / 8;
}

// The sums of a workgroup's v in all its threads, always in the same order.
template <int THREADS, int K>
__device__ inline void add_threads(double (&v)[K]) {
    __shared__ double red[THREADS / 64][K];
#pragma unroll
    for (int k = 0; k < K; ++k)
        for (int off = 1; off < 64; off <<= 1) v[k] += __shfl_xor(v[k], off);
    __syncthreads();                           // of what an earlier call put there, all is read
    if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int k = 0; k < K; ++k) red[threadIdx.x >> 6][k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
        v[k] = 0.0;
#pragma unroll 4
        for (int w = 0; w < THREADS / 64; ++w) v[k] += red[w][k];
    }
}

// Makes the compiler forget what it knows of a register: what follows from it is computed again rather than kept (the
// places of 8 pieces and their widened values would not fit a thread's 128 registers, and went to memory).
template <typename R>
__device__ inline void forget(R& r) { asm volatile("" : "+v"(r)); }

template <typename T>
__device__ inline void forget_raw(typename Pack<T>::raw& r) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    u32x4 v = __builtin_bit_cast(u32x4, r);
    forget(v);
    r = __builtin_bit_cast(typename Pack<T>::raw, v);
}

// The i-th piece of a thread: where it begins, and its first value that is its own (the last piece of a row is moved back
// to end with it; a piece past the end has none and reads the first one).
template <typename T, int THREADS, bool WHOLE>
struct ChannelPieces {
    static constexpr int V = Pack<T>::V;
    uint32_t c, thread, total, stride;
    float per_row;

    __device__ ChannelPieces(const NormParams& p, uint32_t c) : c(c), thread(threadIdx.x) {
        total = (uint32_t)p.n * (uint32_t)p.nvec;
        stride = (uint32_t)p.c * (uint32_t)p.hw;
        per_row = 1.f / (float)p.nvec;
    }
    __device__ bool there(int i) const { return i * THREADS + thread < total; }
    // The row comes from a product: below 8192 pieces it is off by less than the half that keeps it from the next one.
    __device__ size_t place(const NormParams& p, int i, int& own) const {
        const uint32_t piece = there(i) ? i * THREADS + thread : 0, row = (uint32_t)(((float)piece + 0.5f) * per_row);
        const uint32_t begin = (piece - row * (uint32_t)p.nvec) * V, last = (uint32_t)p.hw - V, off = WHOLE || begin < last ? begin : last;
        own = there(i) ? (int)(begin - off) : V;
        return (size_t)row * stride + (c * (uint32_t)p.hw + off);
    }
    __device__ size_t place(const NormParams& p, int i) const {
        int own;
        return place(p, i, own);
    }
    __device__ static bool counts(int own, int k) { return WHOLE ? own == 0 : k >= own; }
};

// 1 / sqrt(v): a root in 32 bits, and one step of Newton's in 64 (every thread needs it, and a division and a root in 64 bits
// are slow); those where 32 bits do not hold the number (an eps of zero and a tiny variance, zero, infinity).
__device__ inline float inverse_root(double v) {
    if (!(v > 1e-36 && v < 1e36)) return (float)(1.0 / sqrt(v));
    const double near = rsqrtf((float)v);
    return (float)(near * (1.5 - 0.5 * v * near * near));
}

// WHOLE: rows are whole pieces.
template <typename T, int THREADS, int PIECES, bool WHOLE>
__global__ __launch_bounds__(THREADS) void k_channel_forward(const T* __restrict__ x, T* __restrict__ out, const NormParams p) {
    constexpr int V = Pack<T>::V;
    const uint32_t c = channel_of(blockIdx.x, gridDim.x);
    ChannelPieces<T, THREADS, WHOLE> q(p, c);
    const float weight = p.weight[c], bias = p.bias[c];
    typename Pack<T>::raw raw[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) raw[i] = load_raw(x + q.place(p, i));
    forget(q.thread);
    double mean, var;
    if (p.training) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            int own;
            q.place(p, i, own);
            const auto v = widen<T>(raw[i]);
#pragma unroll
            for (int k = 0; k < V; ++k) s += q.counts(own, k) ? v[k] : 0.f;
        }
        double first[1] = {s};
        add_threads<THREADS>(first);
        forget(q.thread);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) forget_raw<T>(raw[i]);
        const float about = (float)(first[0] * p.per_count);
        float d1 = 0.f, d2 = 0.f;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            int own;
            q.place(p, i, own);
            const auto v = widen<T>(raw[i]);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float d = q.counts(own, k) ? v[k] - about : 0.f;
                d1 += d;
                d2 += d * d;
            }
        }
        double sums[2] = {d1, d2};
        add_threads<THREADS>(sums);
        forget(q.thread);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) forget_raw<T>(raw[i]);
        const double rest = sums[0] * p.per_count;
        mean = about + rest;
        var = sums[1] * p.per_count - rest * rest;
        if (var < 0.0) var = 0.0;              // a NaN stays one
        if (threadIdx.x == 0) {
            if (p.running_mean) p.running_mean[c] = (float)((1.0 - p.momentum) * p.running_mean[c] + p.momentum * mean);
            if (p.running_var) p.running_var[c] = (float)((1.0 - p.momentum) * p.running_var[c] + p.momentum * var * p.to_sample);
            if (p.num_batches && c == 0) *p.num_batches += 1;
        }
    } else {
        mean = p.running_mean[c];
        var = p.running_var[c];
    }
    const float inv = inverse_root(var + p.eps), m = (float)mean, scale = weight * inv;
    if (threadIdx.x == 0) {
        p.mean[c] = m;
        p.inv[c] = inv;
    }
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        auto v = widen<T>(raw[i]);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = not_below_zero(__builtin_fmaf(v[k] - m, scale, bias));
        if (q.there(i)) store_raw(out + q.place(p, i), v);
    }
}

template <typename T, int THREADS, int PIECES, bool WHOLE>
__global__ __launch_bounds__(THREADS) void k_channel_backward(const T* __restrict__ x, const T* __restrict__ grad, T* __restrict__ dx,
                                                              const NormParams p) {
    constexpr int V = Pack<T>::V;
    const uint32_t c = channel_of(blockIdx.x, gridDim.x);
    ChannelPieces<T, THREADS, WHOLE> q(p, c);
    const float m = p.mean[c], inv = p.inv[c], scale = p.weight[c] * inv, bias = p.bias[c];
    typename Pack<T>::raw raw[PIECES], gr[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const size_t at = q.place(p, i);
        raw[i] = load_raw(x + at);
        gr[i] = load_raw(grad + at);
    }
    forget(q.thread);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        int own;
        q.place(p, i, own);
        const auto v = widen<T>(raw[i]);
        const auto g = widen<T>(gr[i]);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float xc = v[k] - m, gm = q.counts(own, k) && !(__builtin_fmaf(xc, scale, bias) <= 0.f) ? g[k] : 0.f;
            s1 += gm;
            s2 += gm * xc;
        }
    }
    double sums[2] = {s1, s2};
    add_threads<THREADS>(sums);
    forget(q.thread);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        forget_raw<T>(raw[i]);
        forget_raw<T>(gr[i]);
    }
    if (threadIdx.x == 0) {
        p.dbias[c] = (float)sums[0];
        p.dweight[c] = (float)(sums[1] * inv);
    }
    const float b = (float)(-scale * (sums[1] * inv * p.per_count)), d = (float)(-scale * (sums[0] * p.per_count));
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const auto v = widen<T>(raw[i]);
        auto g = widen<T>(gr[i]);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float xc = v[k] - m, gm = __builtin_fmaf(xc, scale, bias) <= 0.f ? 0.f : g[k];
            g[k] = gm * scale + (p.training ? xc * inv * b + d : 0.f);
        }
        if (q.there(i)) store_raw(dx + q.place(p, i), g);
    }
}

// ---------------------------------------------------------------------------------------------- host side
// f(lanes to a row, how the row fits them)
template <typename T, typename F>
static void with_lanes(const NormParams& p, F&& f) {
    constexpr int V = Pack<T>::V;
    typedef std::integral_constant<Fit, EXACT> Exact;
    typedef std::integral_constant<Fit, ONE> One;
    if (p.hw == 8 * V) f(std::integral_constant<int, 8>(), Exact());
    else if (p.hw == 16 * V) f(std::integral_constant<int, 16>(), Exact());
    else if (p.nvec > 64) f(std::integral_constant<int, 64>(), std::integral_constant<Fit, LOOP>());
    else if (p.hw < V) f(std::integral_constant<int, 8>(), std::integral_constant<Fit, LOOP>());
    else if (p.nvec <= 8) f(std::integral_constant<int, 8>(), One());
    else if (p.nvec <= 16) f(std::integral_constant<int, 16>(), One());
    else if (p.nvec <= 32) f(std::integral_constant<int, 32>(), One());
    else f(std::integral_constant<int, 64>(), One());
}

// Whether a workgroup holds a channel.
static bool by_channel(const az_norm_args* a, int nvec, int V) {
    return !a->hidden && !a->channels_last && a->hw >= V && a->n * nvec <= CHANNEL_PIECES && a->c < 1 << 22 &&      // (2^32 threads)
           (int64_t)a->c * a->hw <= 0x7FFFFFFF;
}

// f(threads, pieces a thread, whether rows are whole pieces)
template <typename T, typename F>
static void with_channel(const NormParams& p, F&& f) {
    const auto whole = [&](auto threads, auto pieces) {
        if (p.hw % Pack<T>::V == 0) f(threads, pieces, std::true_type());
        else f(threads, pieces, std::false_type());
    };
    const int64_t pieces = p.n * p.nvec;
    if (pieces <= 1024) whole(std::integral_constant<int, 256>(), std::integral_constant<int, 4>());
    else if (pieces <= 4096) whole(std::integral_constant<int, 1024>(), std::integral_constant<int, 4>());
    else whole(std::integral_constant<int, 1024>(), std::integral_constant<int, 8>());
}

// f(whether the channels are at least one piece of 16 bytes)
template <typename T, typename F>
static void with_pieces(const NormParams& p, F&& f) {
    if (p.c >= Pack<T>::V) f(std::true_type());
    else f(std::false_type());
}

// Which boards a chunk of the pass over the activations holds.
template <typename T>
static void set_chunks(NormParams& p, bool last) {
    p.chunk_boards = p.abreast = 1;
    p.chunks = p.n;
    if (last) return;
    with_lanes<T>(p, [&](auto L, auto) {
        const RowGrid g = row_grid(p, L);
        p.chunk_boards = BOARDS_AT_ONCE;
        p.abreast = (int)g.abreast;
        p.chunks = (int64_t)(g.blocks / g.across) * g.abreast;
    });
}

template <typename T, bool GATED>
static int norm_forward(NormParams p, bool last, const T* x, const T* residual, T* out, hipStream_t s) {
    const int wide = p.nvec < 64 ? p.nvec : 64;
    const dim3 boards((uint32_t)p.n, (p.nvec + wide - 1) / wide), block(NORM_THREADS);
    if (p.by_channel) {
        with_channel<T>(p, [&](auto threads, auto pieces, auto whole) {
            hipLaunchKernelGGL((k_channel_forward<T, decltype(threads)::value, decltype(pieces)::value, decltype(whole)::value>), dim3(p.c), dim3(threads), 0, s, x, out, p);
        });
        AZ_HIP(hipGetLastError());
        return AZ_OK;
    }
    set_chunks<T>(p, last);
    if (p.training || GATED) {
        if (last) with_pieces<T>(p, [&](auto full) { hipLaunchKernelGGL((k_last_stats<T, decltype(full)::value, GATED>), boards, block, 0, s, x, p, wide); });
        else with_lanes<T>(p, [&](auto L, auto fit) {
            const RowGrid g = row_grid(p, L);
            hipLaunchKernelGGL((k_row_stats<T, decltype(L)::value, decltype(fit)::value, GATED>), dim3(g.blocks), block, 0, s, x, p, g);
        });
        AZ_HIP(hipGetLastError());
    }
    hipLaunchKernelGGL(k_channel_stats, dim3((p.c + CHANNELS - 1) / CHANNELS), dim3(CHANNELS * LINES), 0, s, p);
    AZ_HIP(hipGetLastError());
    if (GATED) {
        hipLaunchKernelGGL(k_gate_forward, dim3((uint32_t)((p.n + GATE_ROWS - 1) / GATE_ROWS)), dim3(GATE_THREADS),
                           sizeof(f32x4) * (3 * p.c + p.hidden), s, p);
        AZ_HIP(hipGetLastError());
    }
    if (last) with_pieces<T>(p, [&](auto full) { hipLaunchKernelGGL((k_last_apply<T, decltype(full)::value, GATED>), boards, block, 0, s, x, residual, out, p, wide); });
    else with_lanes<T>(p, [&](auto L, auto fit) {
        const RowGrid g = row_grid(p, L);
        hipLaunchKernelGGL((k_row_apply<T, decltype(L)::value, decltype(fit)::value, GATED>), dim3(g.blocks), block, 0, s, x, residual, out, p, g);
    });
    AZ_HIP(hipGetLastError());
    return AZ_OK;
}

template <typename T, bool GATED>
static int norm_backward(NormParams p, bool last, const T* x, const T* grad, T* dx, T* dresidual, hipStream_t s) {
    const int wide = p.nvec < 64 ? p.nvec : 64;
    const dim3 boards((uint32_t)p.n, (p.nvec + wide - 1) / wide), block(NORM_THREADS);
    if (p.by_channel) {
        with_channel<T>(p, [&](auto threads, auto pieces, auto whole) {
            hipLaunchKernelGGL((k_channel_backward<T, decltype(threads)::value, decltype(pieces)::value, decltype(whole)::value>), dim3(p.c), dim3(threads), 0, s, x, grad, dx, p);
        });
        AZ_HIP(hipGetLastError());
        return AZ_OK;
    }
    set_chunks<T>(p, last);
    if (last) with_pieces<T>(p, [&](auto full) { hipLaunchKernelGGL((k_last_grad_sums<T, decltype(full)::value, GATED>), boards, block, 0, s, x, grad, dresidual, p, wide); });
    else with_lanes<T>(p, [&](auto L, auto fit) {
        const RowGrid g = row_grid(p, L);
        hipLaunchKernelGGL((k_row_grad_sums<T, decltype(L)::value, decltype(fit)::value, GATED>), dim3(g.blocks), block, 0, s, x, grad, dresidual, p, g);
    });
    AZ_HIP(hipGetLastError());
    if (GATED) {
        p.chunks = (p.n + GATE_ROWS - 1) / GATE_ROWS;
        hipLaunchKernelGGL(k_gate_backward, dim3((uint32_t)p.chunks), dim3(GATE_THREADS),
                           sizeof(f32x4) * (2 * p.c + p.hidden + GATE_THREADS * 4), s, p);
        AZ_HIP(hipGetLastError());
    }
    const int cb = (p.c + CHANNELS - 1) / CHANNELS;
    hipLaunchKernelGGL(k_param_grads, dim3(cb + (GATED ? weight_tiles(p) * weight_splits(p) : 0)), dim3(CHANNELS * LINES), 0, s, p, cb);
    AZ_HIP(hipGetLastError());
    const T* masked = GATED ? dresidual : grad;
    const uint32_t joins = (uint32_t)join_blocks(p);
    if (last) with_pieces<T>(p, [&](auto full) { hipLaunchKernelGGL((k_last_grad_apply<T, decltype(full)::value, GATED>), dim3(boards.x + joins, boards.y), block, 0, s, x, masked, dx, p, wide, joins); });
    else with_lanes<T>(p, [&](auto L, auto fit) {
        const RowGrid g = row_grid(p, L);
        hipLaunchKernelGGL((k_row_grad_apply<T, decltype(L)::value, decltype(fit)::value, GATED>), dim3(g.blocks + joins), block, 0, s, x, masked, dx, p, g, joins);
    });
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
    const int nvec = (int)(((int64_t)(a->channels_last ? a->c : a->hw) + V - 1) / V);
    const int64_t groups = nvec <= 8 ? 32 : nvec <= 16 ? 16 : nvec <= 32 ? 8 : 4, room = MOST_BLOCKS - 16384;      // (the weights' joins)
    AZ_CHECK_ARG(a->channels_last ? a->n <= room && a->c <= 1 << 23 : (a->n + 3) / 4 * ((a->c + groups - 1) / groups) <= room && a->c < 1 << 26,
                 "norm: %lld x %d x %d is more than a launch takes", (long long)a->n, a->c, a->hw);
    const size_t rows = (size_t)a->n * a->c, hidden = (size_t)a->n * a->hidden;
    p->n = a->n;
    p->c = a->c;
    p->hw = a->hw;
    p->hidden = a->hidden;
    p->nvec = nvec;
    p->training = a->training != 0;
    p->eps = a->eps;
    p->momentum = a->momentum;
    p->per_count = 1.0 / ((double)a->n * a->hw);
    p->to_sample = 1.0 / (1.0 - p->per_count);
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
    p->board_mean = p->gate = p->h = p->s1 = p->s2 = p->de = p->dh = p->dq = p->partial = nullptr;
    p->mean = saved.take<float>(a->c);
    p->inv = saved.take<float>(a->c);
    p->by_channel = by_channel(a, nvec, V);
    if (p->by_channel) {                      // nothing else is kept, and no workspace used
        p->mask = nullptr;
        p->part_a = p->part_b = p->A = p->B = p->ca = p->cb = p->cd = nullptr;
        if (sizes) {
            sizes[0] = (int64_t)saved.used;
            sizes[1] = sizes[2] = 0;
        }
        return AZ_OK;
    }
    if (a->hidden) {
        p->board_mean = saved.take<float>(rows);
        p->gate = saved.take<float>(rows);
        p->h = saved.take<float>(hidden);
    }
    p->mask = saved.take<uint8_t>((size_t)p->nvec * (a->channels_last ? (size_t)a->n * a->hw : rows));
    // both passes begin with the partial sums: at most one chunk per board, and a row more per board that lies abreast
    p->part_a = fwd.take<float>(rows + (size_t)NORM_THREADS * a->c);
    p->part_b = fwd.take<float>(rows + (size_t)NORM_THREADS * a->c);
    bwd.used = fwd.used;
    p->A = fwd.take<float>(a->hidden ? rows : a->c);
    p->B = fwd.take<float>(a->hidden ? rows : a->c);
    p->ca = bwd.take<float>(a->c);
    p->cb = bwd.take<float>(a->c);
    p->cd = bwd.take<float>(a->c);
    if (a->hidden) {
        p->s1 = bwd.take<float>(rows);
        p->s2 = bwd.take<float>(rows);
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

static int norm_check(const az_norm_args* a, const NormParams& p) {
    AZ_CHECK_ARG(a->x_dev && a->weight_dev && a->bias_dev && a->saved_dev && (a->workspace_dev || p.by_channel), "norm: null argument");
    AZ_CHECK_ARG((uintptr_t)a->saved_dev % 16 == 0 && (uintptr_t)a->workspace_dev % 16 == 0, "norm: buffers must be 16-byte aligned");
    AZ_CHECK_ARG(!a->hidden || (a->fc1_weight_dev && a->fc1_bias_dev && a->fc2_weight_dev && a->fc2_bias_dev), "norm: null gate weights");
    return AZ_OK;
}

// f(a value of the activations' type, whether there is a gate)
template <typename F>
static int with_type(const az_norm_args* a, F&& f) {
    const auto gated = [&](auto t) { return a->hidden ? f(t, std::true_type()) : f(t, std::false_type()); };
    return a->dtype == AZ_F32 ? gated(0.f) : a->dtype == AZ_BF16 ? gated((__bf16)0.f) : gated((_Float16)0.f);
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
    if (rc == AZ_OK) rc = norm_check(a, p);
    if (rc != AZ_OK) return rc;
    AZ_CHECK_ARG(a->out_dev && (!a->hidden || a->residual_dev), "az_norm_forward: null argument");
    AZ_CHECK_ARG(a->training || (a->running_mean_dev && a->running_var_dev), "az_norm_forward: evaluation without running statistics");
    return with_type(a, [&](auto t, auto gated) {
        typedef decltype(t) T;
        return norm_forward<T, decltype(gated)::value>(p, a->channels_last != 0, (const T*)a->x_dev, (const T*)a->residual_dev, (T*)a->out_dev,
                                                       (hipStream_t)stream);
    });
}

extern "C" int az_norm_backward(const az_norm_args* a, void* stream) {
    NormParams p;
    int rc = norm_params(a, &p, nullptr);
    if (rc == AZ_OK) rc = norm_check(a, p);
    if (rc != AZ_OK) return rc;
    AZ_CHECK_ARG(a->grad_dev && a->dx_dev && a->dweight_dev && a->dbias_dev, "az_norm_backward: null argument");
    AZ_CHECK_ARG(!a->hidden || (a->dresidual_dev && a->dfc1_weight_dev && a->dfc1_bias_dev && a->dfc2_weight_dev && a->dfc2_bias_dev),
                 "az_norm_backward: null gate gradient");
    return with_type(a, [&](auto t, auto gated) {
        typedef decltype(t) T;
        return norm_backward<T, decltype(gated)::value>(p, a->channels_last != 0, (const T*)a->x_dev, (const T*)a->grad_dev, (T*)a->dx_dev,
                                                        (T*)a->dresidual_dev, (hipStream_t)stream);
    });
}
