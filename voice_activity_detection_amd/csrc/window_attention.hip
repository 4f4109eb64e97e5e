// Attention with a sliding window and sinks: row i of a sequence sees key j when j <= i and (i - j < window or j < sinks).
//
//   P = softmax over the visible keys of scale q k^T,  O = P V
//   dV = P^T dO,  dS = P (dO V^T - rowsum(dO O)),  dQ = scale dS K,  dK = scale dS^T Q
//
// Every kernel keeps rows of one side in registers (queries for O and dQ, keys for dK and dV) and streams tiles of 64
// rows of the other side through LDS, visiting only tiles that some row of the block sees.  Scores are formed
// transposed -- own rows along the lanes, streamed rows down the result tile -- so that the softmax of a row stays
// within four lanes and the weights are, without moving, the operand of the second product.  The forward pass goes over
// the keys once with a running maximum and sum, and keeps (maximum, 1 / sum) per row for the backward pass, both in
// float32 and in units of log2.
//
// Key heads shared by several query heads: the forward pass and dQ run per query head, dK and dV add their query heads
// in registers.  The few sink keys are seen by every later row; their share of dK and dV is a second kernel over
// segments of the rows, joined in a fixed order.
//
// Bound by matrix products, the exponentials beside them and, in dK and dV of 64 columns, the reads of tiles from LDS.  Measured,
// bfloat16: 2 x 16 heads of 128 over 8192 rows, window 1000, O in 213 us (590 TFLOP/s of visible pairs); 8 ragged sequences of
// up to 2000 rows, 8 query heads of 64 on 2 key heads, window 300: O 36, dQ 55, dK and dV 60, those of 4 sinks 11 + 7 us.  The
// step reads its cache once and is bound by that: 32 x 4 heads of 4004 slots of 128, 262 MB in 59 us (4.5 TB/s), 5 us for the
// join of its splits.  (Passes in a row; the comparisons beside the choices below were taken in turn on a card that had just been
// idle, where the same kernels are up to a sixth slower.)
//
// A row outside a key's window must not feel what that key holds.  Scores are replaced, not multiplied, where the mask
// says so.  Where a partly visible tile holds an infinity or a NaN, which the matrix product would multiply by zero, it is
// taken out of the tile once the scores are formed.  A visible one still reaches its rows: through a weight that its own
// score has made NaN, or, where no score depends on it (V in O, dO in dV) or the score may be minus infinity and its weight
// zero (K in dQ), by a pass over the block's outputs at its end, which costs a block that meets one a walk over its
// window (0.6 ms at 1000 rows, 6 ms at 8192) and the others nothing.

#include <mutex>
#include <type_traits>

#include "sequence_device.h"

namespace vad {
namespace {
using namespace sq;

constexpr int kTile = 64;           // streamed rows
constexpr int kThreads = 256;

template <typename T>
struct WindowArgs {
    Heads<const T> q, k, v, go;
    const T* o;                     // outputs of the forward pass (backward)
    T* out;                         // o, or dq
    T* dk;
    T* dv;
    float* stats;                   // (row, head): maximum, 1 / sum
    float* delta;                   // (row, head): rowsum(dO O)
    float* parts;                   // (seq, kv head, 1 + segments, dk | dv, sinks, dim)
    Sequences seq;
    int n_seq, heads, kv_heads, dim, window, sinks, segments;
    unsigned tiles;                 // blocks per head and sequence
    float scale;
    bool whole;                     // all rows are whole words at 4-byte boundaries
};

// A block's LDS: tiles of two tensors, twice where that leaves room for two blocks on a compute unit -- the next tiles are
// then written while the present ones are read, with one barrier between tiles instead of two.
template <typename T, int DP>
struct TileShape {
    // The padding spreads the banks (64 of 4 bytes): eight rows' 16-byte pieces at one column, and as many rows' 32-byte
    // pieces as the transposing read takes them, fall into different ones.  (64 columns of bfloat16 would want 16 elements
    // as well, but with 8 a fourth block fits the compute unit's LDS: 291 against 335 us on 4 x 16 heads of 8192 rows.)
    static constexpr int kLd = DP + (sizeof(T) == 4 ? 4 : (DP == 64 ? 8 : 16));
    static constexpr int kTileElems = kTile * kLd;
    static constexpr int kBuffers = 4 * kTileElems * sizeof(T) <= 72 * 1024 ? 2 : 1;
    static constexpr int kExtra = 3 * kTile;          // floats per buffer beside the tiles
    static constexpr size_t lds(int buffers) { return (size_t)buffers * (2 * kTileElems * sizeof(T) + kExtra * sizeof(float)) + 4 * sizeof(int); }
};

// Own rows first .. first + 64 NB - 1 of a head (zero from row `len` on) as fragments: requested early, then by way of the
// block's first two tiles.
template <typename T, int DP, int NB, int NT, bool BUF>
struct Own {
    static constexpr int kLd = TileShape<T, DP>::kLd;
    Staged<T, DP, NT, BUF, kLd> r[NB];
    __device__ __forceinline__ void fetch(const T* p, int64_t st, int first, int len, int dim) {
#pragma unroll
        for (int n = 0; n < NB; ++n) r[n].fetch(p, st, first + 64 * n, len - first - 64 * n, dim);
    }
    __device__ __forceinline__ void take(Frag<T> (&f)[NB][DP / 32], T* tiles, int dim) {
        const int wave = threadIdx.x >> 6;
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NB; ++n) r[n].put(tiles + n * kTile * kLd, dim);
        __syncthreads();
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) f[nb][d] = frag_natural(tiles, kLd, 16 * (NB * wave + nb), 32 * d);
    }
};

// acc (columns of the tile down, own rows along the lanes) += tile^T p, p the weights of 16 KB streamed rows for this lane's
// own row.
template <typename T, int DP, int NB, int KB>
__device__ __forceinline__ void accumulate(const T* tile, const f32x4 (&p)[KB][NB], f32x4 (&acc)[DP / 16][NB]) {
#pragma unroll
    for (int t = 0; t < KB / 2; ++t) {
        Frag<T> f[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) to_frag(p[2 * t][nb], p[2 * t + 1][nb], f[nb]);
#pragma unroll
        for (int b = 0; b < DP / 16; ++b) {
            const Frag<T> x = frag_columns(tile, TileShape<T, DP>::kLd, 32 * t, 16 * b);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) acc[b][nb] = mma(x, f[nb], acc[b][nb]);
        }
    }
}

// The same for two sets of weights, each piece of the tile read once.
template <typename T, int DP, int NB, int KB>
__device__ __forceinline__ void accumulate(const T* tile, const f32x4 (&p)[KB][NB], f32x4 (&acc)[DP / 16][NB], const f32x4 (&p2)[KB][NB],
                                           f32x4 (&acc2)[DP / 16][NB]) {
#pragma unroll
    for (int t = 0; t < KB / 2; ++t) {
        Frag<T> f[NB], f2[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            to_frag(p[2 * t][nb], p[2 * t + 1][nb], f[nb]);
            to_frag(p2[2 * t][nb], p2[2 * t + 1][nb], f2[nb]);
        }
#pragma unroll
        for (int b = 0; b < DP / 16; ++b) {
            const Frag<T> x = frag_columns(tile, TileShape<T, DP>::kLd, 32 * t, 16 * b);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                acc[b][nb] = mma(x, f[nb], acc[b][nb]);
                acc2[b][nb] = mma(x, f2[nb], acc2[b][nb]);
            }
        }
    }
}

// What the infinities and NaN of rows [i0, i1) of a column add up to; zero where there are none.
template <typename T>
__device__ __forceinline__ float not_finite_sum(const T* p, int64_t st, int64_t i0, int64_t i1) {
    float sum = 0.0f;
#pragma unroll 8
    for (int64_t i = i0; i < i1; ++i) {
        const float x = (float)p[i * st];
        sum += fabsf(x) < INFINITY ? 0.0f : x;
    }
    return sum;
}

// s = tile own^T for 16 KB streamed rows
template <typename T, int DP, int NB, int KB>
__device__ __forceinline__ void scores(const T* tile, const Frag<T> (&own)[NB][DP / 32], f32x4 (&s)[KB][NB]) {
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) s[kb][nb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) {
            const Frag<T> x = frag_natural(tile, TileShape<T, DP>::kLd, 16 * kb, 32 * d);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) s[kb][nb] = mma(x, own[nb][d], s[kb][nb]);
        }
    }
}

// The key tiles that rows r0 .. r1 see: the first sink tile if it lies before the band, then the band's.
struct KeyTiles {
    int band, end;                  // first rows of the band's first tile, and past its last
    bool sink;
    __device__ __forceinline__ KeyTiles(int r0, int r1, int window, int sinks) {
        const int lo = r0 - window + 1;
        band = lo > 0 ? lo / kTile * kTile : 0;
        end = r1 / kTile * kTile + kTile;
        sink = sinks > 0 && band > 0;
    }
    __device__ __forceinline__ int first() const { return sink ? 0 : band; }
    __device__ __forceinline__ int next(int t) const { return sink && t == 0 ? band : t + kTile; }
};

// A launch's blocks are dealt to the eight dies in turn; this gives each die a contiguous range of the work, so that
// neighbouring tiles and the query heads of a key head meet in one L2.
__device__ __forceinline__ unsigned work_index() {
    const unsigned n = gridDim.x, die = blockIdx.x % 8, rest = n % 8;
    return die * (n / 8) + (die < rest ? die : rest) + blockIdx.x / 8;
}

// BACK == false: O and stats.  BACK == true: dQ and delta.
template <typename T, int DP, int NB, bool BACK, bool BUF>
__global__ __launch_bounds__(kThreads, 2) void window_rows_kernel(WindowArgs<T> a) {
    using C = TileShape<T, DP>;
    extern __shared__ char lds_raw[];
    T* tiles = reinterpret_cast<T*>(lds_raw);             // K and V, once or twice
    int* flags = reinterpret_cast<int*>(tiles + 2 * C::kBuffers * C::kTileElems);
    const unsigned work = work_index();
    const int part = work % a.tiles, h = work / a.tiles % a.heads, s = work / a.tiles / a.heads, hk = h / (a.heads / a.kv_heads);
    int64_t first, len64;
    sequence_rows(a.seq, s, first, len64);
    const int len = (int)len64, dim = a.dim;
    const int lane = lane_id(), wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    const T* qp = head_ptr(a.q, a.seq, s, first, h);
    const T* kp = head_ptr(a.k, a.seq, s, first, hk);
    const T* vp = head_ptr(a.v, a.seq, s, first, hk);
    const T* gp = BACK ? head_ptr(a.go, a.seq, s, first, h) : nullptr;
    const int64_t row_base = a.seq.starts ? first : (int64_t)s * a.seq.max_len;
    const float l2scale = a.scale * kLog2e;
    constexpr int kRows = 64 * NB;
    // delta of bfloat16 outputs is off by their rounding and that of the weights behind them, 2^-8 of dO O, which is not small
    // beside dP - delta where few keys share a row.  The sum of a row's dS tells by how much, and dQ is off by that times the
    // mean key: one more product, 50 -> 62 us on 8 ragged sequences of up to 2000 rows (8 heads of 64, window 300), for gradients
    // at 2^-8.7 of the exact ones in place of 2^-7.8 (window 2) and 2^-8.5 (window 300).
    constexpr bool kRefine = BACK && sizeof(T) == 2;
    // with 128 columns half a tile's scores at a time, or registers run out: 463 -> 420 us on 2 x 16 heads of 8192 rows, window 1000
    // (64 columns: 456 -> 466 us on twice the sequences, 32: 274 -> 289)
    constexpr int kHalves = kRefine && DP == 128 ? 2 : 1, kPart = kTile / kHalves;
    zero_outside(a.out, (int64_t)a.heads * dim, h * dim, dim, a.seq, s, a.n_seq, part, a.tiles);
    // flags[turn]: the tile in hand holds infinities or NaN; the next tile's is set and the last one's cleared meanwhile
    if (threadIdx.x < 3) flags[threadIdx.x] = 0;
    int turn = 0, buffer = 0;
    bool met = false;
    for (int64_t r0_64 = (int64_t)part * kRows; r0_64 < len; r0_64 += (int64_t)a.tiles * kRows) {
        const int r0 = (int)r0_64, r1 = (len - r0 < kRows ? len - r0 : kRows) + r0 - 1;
        const int w0 = r0 + 16 * NB * wave, w1 = w0 + 16 * NB - 1;
        Frag<T> qf[NB][DP / 32], gf[NB][DP / 32];
        f32x4 acc[DP / 16][NB], mean[DP / 16][NB];
        float m[NB], sum[NB], delta[NB], off[NB];
        const KeyTiles keys(r0, r1, a.window, a.sinks);
        Staged<T, DP, kThreads, BUF, C::kLd> rk, rv;
        const auto fetch = [&](int t) {
            const int left = t < keys.end ? len - t : 0;       // no branch: no rows behind the last tile
            rk.fetch(kp, a.k.st, t, left, dim);
            rv.fetch(vp, a.v.st, t, left, dim);
        };
        Own<T, DP, NB, kThreads, BUF> own_q;
        own_q.fetch(qp, a.q.st, r0, len, dim);
        if (BACK) {
            Own<T, DP, NB, kThreads, BUF> own_g, own_o;
            own_g.fetch(gp, a.go.st, r0, len, dim);
            own_o.fetch(a.o + (row_base * a.heads + h) * dim, (int64_t)a.heads * dim, r0, len, dim);
            fetch(keys.first());
            Frag<T> of[NB][DP / 32];
            own_q.take(qf, tiles, dim);
            own_g.take(gf, tiles, dim);
            own_o.take(of, tiles, dim);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                float x = 0.0f;
#pragma unroll
                for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                    for (int j = 0; j < 8; ++j) x = fmaf((float)gf[nb][d][j], (float)of[nb][d][j], x);
                delta[nb] = groups_sum(x);
            }
        } else {
            fetch(keys.first());
            own_q.take(qf, tiles, dim);
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int row = w0 + 16 * nb + c;
            const bool live = row < len;
            m[nb] = -INFINITY;
            sum[nb] = 0.0f;
            if (BACK) {
                const int64_t at = (row_base + row) * a.heads + h;
                m[nb] = live ? a.stats[2 * at] : 0.0f;
                sum[nb] = live ? a.stats[2 * at + 1] : 0.0f;
            }
            off[nb] = 0.0f;
#pragma unroll
            for (int b = 0; b < DP / 16; ++b) acc[b][nb] = mean[b][nb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        const auto is_edge = [&](int t) { return !(t + kTile - 1 <= r0 && r0 + kRows - 1 - t < a.window); };
        const auto put = [&](int t, int to, int flag) {
            rk.put(tiles + 2 * to * C::kTileElems, dim);
            rv.put(tiles + (2 * to + 1) * C::kTileElems, dim);
            if (is_edge(t) && (BACK ? rk : rv).not_finite()) flags[flag] = 1;
        };
        __syncthreads();                                       // the own rows' fragments are read
        if (C::kBuffers == 2) {
            put(keys.first(), buffer, turn);
            fetch(keys.next(keys.first()));
            __syncthreads();
        }
        for (int t = keys.first(); t < keys.end; t = keys.next(t)) {
            const int nt = keys.next(t), after = turn == 2 ? 0 : turn + 1;
            if (C::kBuffers == 2) {
                put(nt, buffer ^ 1, after);
                fetch(keys.next(nt));
            } else {
                if (t != keys.first()) __syncthreads();
                put(t, 0, turn);
                __syncthreads();
                fetch(nt);
            }
            T* sk = tiles + 2 * buffer * C::kTileElems;
            T* sv = sk + C::kTileElems;
            // EDGE: some row of the block does not see all of the tile
            const auto step = [&](auto edge) {
            constexpr bool EDGE = decltype(edge)::value;
            const bool active = !EDGE || (t <= w1 && (w0 - (t + kTile - 1) < a.window || t < a.sinks));      // for this wave
#pragma unroll 1
            for (int half = 0; half < kHalves; ++half) {
            T* pk = sk + half * kPart * C::kLd;
            T* pv = sv + half * kPart * C::kLd;
            f32x4 p[kPart / 16][NB], dp[kPart / 16][NB];
            if (active) {
                // products ahead of the other waves' softmax: 228 -> 223 us at 128 columns, 299 -> 295 at 64
                __builtin_amdgcn_s_setprio(1);
                scores<T, DP, NB>(pk, qf, p);
                if (BACK) scores<T, DP, NB>(pv, gf, dp);
                __builtin_amdgcn_s_setprio(0);
            }
            if (EDGE && flags[turn]) {
                __syncthreads();
                clean_tile<T, DP, kThreads, C::kLd>(BACK ? pk : pv, kPart);
                __syncthreads();
                met = true;
            }
            if (active) {
            const bool masked = EDGE && !(t + kTile - 1 <= w0 && w1 - t < a.window);
            if (masked) {
#pragma unroll
                for (int kb = 0; kb < kPart / 16; ++kb)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int j = t + half * kPart + 16 * kb + 4 * g + i, gap = w0 + 16 * nb + c - j;
                            const bool sees = ((unsigned)gap < (unsigned)a.window) | ((gap >= 0) & (j < a.sinks));
                            p[kb][nb][i] = sees ? p[kb][nb][i] : -INFINITY;
                        }
            }
            if (!BACK) {
                // The running maximum follows only where the weights would pass 2^8: the sums are the same, and the outputs
                // are rescaled a few times per row instead of at every tile.
                float top[NB];
                bool grow = false;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    top[nb] = p[0][nb][0];
#pragma unroll
                    for (int kb = 0; kb < kPart / 16; ++kb)
#pragma unroll
                        for (int i = 0; i < 4; ++i) top[nb] = fmaxf(top[nb], p[kb][nb][i]);
                    top[nb] = groups_max(top[nb]) * l2scale;
                    grow |= top[nb] > m[nb] + 8.0f;
                }
                if (__any(grow)) {
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        const float now = fmaxf(m[nb], top[nb]);
                        const float shrink = __builtin_amdgcn_exp2f(m[nb] - (now == -INFINITY ? 0.0f : now));
                        m[nb] = now;
                        sum[nb] *= shrink;
#pragma unroll
                        for (int b = 0; b < DP / 16; ++b) acc[b][nb] *= shrink;
                    }
                }
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    const float base = m[nb] == -INFINITY ? 0.0f : m[nb];
                    float part = 0.0f;
#pragma unroll
                    for (int kb = 0; kb < kPart / 16; ++kb)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            p[kb][nb][i] = __builtin_amdgcn_exp2f(fmaf(p[kb][nb][i], l2scale, -base));
                            part += p[kb][nb][i];
                        }
                    sum[nb] += part;
                }
                __builtin_amdgcn_s_setprio(1);
                accumulate<T, DP, NB>(pv, p, acc);
                __builtin_amdgcn_s_setprio(0);
            } else {
#pragma unroll
                for (int kb = 0; kb < kPart / 16; ++kb)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float x = __builtin_amdgcn_exp2f(fmaf(p[kb][nb][i], l2scale, -m[nb])) * sum[nb];
                            const float y = (p[kb][nb][i] == -INFINITY) & masked ? 0.0f : x * (dp[kb][nb][i] - delta[nb]);
                            if (kRefine) {
                                p[kb][nb][i] = x;
                                off[nb] += y;
                            }
                            dp[kb][nb][i] = y * a.scale;
                        }
                if (kRefine)
                    accumulate<T, DP, NB>(pk, dp, acc, p, mean);
                else
                    accumulate<T, DP, NB>(pk, dp, acc);
            }
            }
            }
            };
            // (the forward pass is faster with one body that asks: 256 against 325 us on 2 x 16 heads of 8192 rows of 128)
            if (!BACK || is_edge(t))
                step(std::true_type{});
            else
                step(std::false_type{});
            if (threadIdx.x == 0) flags[after == 2 ? 0 : after + 1] = 0;
            turn = after;
            if (C::kBuffers == 2) {
                buffer ^= 1;
                __syncthreads();
            }
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int row = w0 + 16 * nb + c;
            const int64_t at = (row_base + row) * a.heads + h;
            float f = 1.0f;
            if (!BACK) {
                f = 1.0f / groups_sum(sum[nb]);
                if (a.stats && row < len && g == 0) {
                    a.stats[2 * at] = m[nb];
                    a.stats[2 * at + 1] = f;
                }
            }
            if (BACK) {
                if (kRefine) {
                    off[nb] = groups_sum(off[nb]);
                    const float back = off[nb] * a.scale;
#pragma unroll
                    for (int b = 0; b < DP / 16; ++b) acc[b][nb] -= mean[b][nb] * back;
                }
                if (row < len && g == 0) a.delta[at] = delta[nb] + off[nb];
            }
            if (row < len) {
#pragma unroll
                for (int b = 0; b < DP / 16; ++b) store_quad(a.out + at * dim, 16 * b + 4 * g, dim, acc[b][nb] * f, BUF);
            }
        }
        if (met) {
            __syncthreads();
            const T* p = BACK ? kp : vp;
            const int64_t st = BACK ? a.k.st : a.v.st;
            for (int e = threadIdx.x; e < (r1 - r0 + 1) * dim; e += kThreads) {
                const int row = r0 + e / dim, d = e % dim, lo = row - a.window + 1 > 0 ? row - a.window + 1 : 0;
                const float x = not_finite_sum(p + d, st, lo, (int64_t)row + 1) + not_finite_sum(p + d, st, 0, lo < a.sinks ? lo : a.sinks);
                T* o = a.out + ((row_base + row) * a.heads + h) * dim + d;
                // dS of such a key is zero or NaN, and so dS K is NaN
                if (x != 0.0f) *o = BACK ? (T)NAN : (T)((float)*o + x);
            }
            met = false;
        }
    }
}

// dK and dV.  SINKS == false: the block's keys against the rows of their window.  SINKS == true: the sink keys against the
// rows beyond their window, one segment of the rows.
//
// The sink keys are few: there a block is one wave with 16 of them, against one segment of the rows of one query head.
template <typename T, int DP, int NB, bool SINKS, bool BUF>
__global__ __launch_bounds__(SINKS ? 64 : kThreads, DP == 128 && (SINKS || sizeof(T) == 4) ? 1 : 2) void window_keys_kernel(WindowArgs<T> a) {
    constexpr int NT = SINKS ? 64 : kThreads;
    using C = TileShape<T, DP>;
    extern __shared__ char lds_raw[];
    constexpr int kBuffers = SINKS ? 1 : C::kBuffers;
    T* tiles = reinterpret_cast<T*>(lds_raw);                                    // Q and dO, once or twice
    float* extras = reinterpret_cast<float*>(tiles + 2 * kBuffers * C::kTileElems);      // maximum, 1 / sum, delta of their rows
    int* flags = reinterpret_cast<int*>(extras + kBuffers * C::kExtra);
    const unsigned work = work_index();
    const int part = work % a.tiles, hk = work / a.tiles % a.kv_heads, s = work / a.tiles / a.kv_heads, group = a.heads / a.kv_heads;
    const int segment = SINKS ? part % a.segments : 0;
    int64_t first, len64;
    sequence_rows(a.seq, s, first, len64);
    const int len = (int)len64, dim = a.dim;
    const int lane = lane_id(), wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    const T* kp = head_ptr(a.k, a.seq, s, first, hk);
    const T* vp = head_ptr(a.v, a.seq, s, first, hk);
    const int64_t row_base = a.seq.starts ? first : (int64_t)s * a.seq.max_len;
    // sink keys' sums go to the joining kernel in float32: [0] those of their window, [1 + n] of segment n
    float* parts = a.parts + (((int64_t)s * a.kv_heads + hk) * (1 + a.segments) + (SINKS ? 1 + segment : 0)) * 2 * a.sinks * dim;
    const float l2scale = a.scale * kLog2e;
    constexpr int kKeys = NT / 4 * NB;
    if (!SINKS) {
        zero_outside(a.dk, (int64_t)a.kv_heads * dim, hk * dim, dim, a.seq, s, a.n_seq, part, a.tiles);
        zero_outside(a.dv, (int64_t)a.kv_heads * dim, hk * dim, dim, a.seq, s, a.n_seq, part, a.tiles);
    }
    if (threadIdx.x < 3) flags[threadIdx.x] = 0;
    int turn = 0, buffer = 0;
    bool met = false;
    // (the sink keys' blocks take one turn)
    for (int64_t j0_64 = (SINKS ? part / a.segments : (int64_t)part) * kKeys; j0_64 < len; j0_64 += SINKS ? len : (int64_t)a.tiles * kKeys) {
        const int j0 = (int)j0_64;
        const int w0 = j0 + 16 * NB * wave, w1 = w0 + 16 * NB - 1;
        // the rows [i0, i1) that see the keys
        int i0 = j0, i1;
        if (SINKS) {
            const int beyond = len > a.window ? len - a.window : 0, cuts = a.segments / group;
            const int per = ((beyond + cuts - 1) / cuts + kTile - 1) / kTile * kTile;
            const int64_t lo = a.window + (int64_t)(segment / group) * per;
            i0 = (int)(lo < len ? lo : len);
            i1 = (int)(lo + per < len ? lo + per : len);
        } else {
            const int64_t hi = (int64_t)j0 + kKeys - 1 + a.window;
            i1 = (int)(hi < len ? hi : len);
        }
        const int keys = SINKS ? (a.sinks < len ? a.sinks : len) : len;
        Frag<T> kf[NB][DP / 32], vf[NB][DP / 32];
        f32x4 dk[DP / 16][NB], dv[DP / 16][NB];
        Own<T, DP, NB, NT, BUF> own_k, own_v;
        own_k.fetch(kp, a.k.st, j0, keys, dim);
        if (!SINKS) own_v.fetch(vp, a.v.st, j0, keys, dim);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int b = 0; b < DP / 16; ++b) dk[b][nb] = dv[b][nb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        const int n_tiles = i1 > i0 ? (i1 - i0 + kTile - 1) / kTile : 0;
        Staged<T, DP, NT, BUF, C::kLd> rq, rg;
        float rm = 0.0f, rinv = 0.0f, rdelta = 0.0f;          // of row threadIdx.x of the tile
        const int h0 = hk * group + (SINKS ? segment % group : 0), heads = SINKS ? 1 : group, steps = n_tiles * heads;
        const auto row_of = [&](int step) { return i0 + step % n_tiles * kTile; };
        const auto fetch = [&](int step) {
            if (step >= steps) return;
            const int h = h0 + step / n_tiles, t = row_of(step);
            rq.fetch(head_ptr(a.q, a.seq, s, first, h), a.q.st, t, i1 - t, dim);
            rg.fetch(head_ptr(a.go, a.seq, s, first, h), a.go.st, t, i1 - t, dim);
            const int row = t + threadIdx.x;
            if (threadIdx.x < kTile) {
                const int64_t at = (row_base + row) * a.heads + h;
                rm = row < i1 ? a.stats[2 * at] : 0.0f;
                rinv = row < i1 ? a.stats[2 * at + 1] : 0.0f;
                rdelta = row < i1 ? a.delta[at] : 0.0f;
            }
        };
        const auto is_edge = [&](int t) { return SINKS || !(t >= j0 + kKeys - 1 && t + kTile - 1 - j0 < a.window && t + kTile <= i1 && j0 + kKeys <= keys); };
        const auto put = [&](int step, int to, int flag) {
            if (step >= steps) return;
            rq.put(tiles + 2 * to * C::kTileElems, dim);
            rg.put(tiles + (2 * to + 1) * C::kTileElems, dim);
            if (threadIdx.x < kTile) {
                float* e = extras + to * C::kExtra + threadIdx.x;
                e[0] = rm;
                e[kTile] = rinv;
                e[2 * kTile] = rdelta;
            }
            if (is_edge(row_of(step)) && (rq.not_finite() || rg.not_finite())) flags[flag] = 1;
        };
        if (!SINKS) fetch(0);
        own_k.take(kf, tiles, dim);
        if (SINKS) own_v.fetch(vp, a.v.st, j0, keys, dim);     // one wave stages whole tiles: one of them at a time in its registers
        own_v.take(vf, tiles, dim);
        __syncthreads();                                       // the own rows' fragments are read
        if (kBuffers == 2) {
            put(0, buffer, turn);
            fetch(1);
            __syncthreads();
        }
        for (int step = 0; step < steps; ++step) {
            const int t = row_of(step), after = turn == 2 ? 0 : turn + 1;
            if (kBuffers == 2) {
                put(step + 1, buffer ^ 1, after);
                fetch(step + 2);
            } else {
                if (SINKS) fetch(step);                        // one wave: its registers hold no tile ahead, other blocks hide the wait
                if (step) __syncthreads();
                put(step, 0, turn);
                __syncthreads();
                if (!SINKS) fetch(step + 1);
            }
            T* sqr = tiles + 2 * buffer * C::kTileElems;
            T* sgo = sqr + C::kTileElems;
            const float* sm = extras + buffer * C::kExtra;
            const float* sinv = sm + kTile;
            const float* sdelta = sinv + kTile;
            const auto work_on = [&](auto edge) {
            constexpr bool EDGE = decltype(edge)::value;
            const bool active = !EDGE || (w0 < keys && (SINKS || (t + kTile - 1 >= w0 && t - w1 < a.window)));
            f32x4 p[4][NB], dp[4][NB];
            if (active) {
                scores<T, DP, NB>(sqr, kf, p);
                scores<T, DP, NB>(sgo, vf, dp);
            }
            if (EDGE && flags[turn]) {
                __syncthreads();
                clean_tile<T, DP, NT, C::kLd>(sqr, kTile);
                clean_tile<T, DP, NT, C::kLd>(sgo, kTile);
                __syncthreads();
                met = true;
            }
            if (active) {
            const auto sees = [&](int row, int nb) {
                const int i = t + row, j = w0 + 16 * nb + c;
                return (i < i1) & (SINKS ? (j < keys) & (i - j >= a.window) : (unsigned)(i - j) < (unsigned)a.window);
            };
            const bool masked = EDGE && (SINKS || !(t >= w1 && t + kTile - 1 - w0 < a.window && t + kTile <= i1));
#pragma unroll
            for (int kb = 0; kb < 4; ++kb) {
                const f32x4 mm = *reinterpret_cast<const f32x4*>(sm + 16 * kb + 4 * g);
                const f32x4 inv = *reinterpret_cast<const f32x4*>(sinv + 16 * kb + 4 * g);
                const f32x4 dl = *reinterpret_cast<const f32x4*>(sdelta + 16 * kb + 4 * g);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const bool see = !masked | sees(16 * kb + 4 * g + i, nb);
                        const float x = __builtin_amdgcn_exp2f(fmaf(p[kb][nb][i], l2scale, -mm[i])) * inv[i];
                        p[kb][nb][i] = see ? x : 0.0f;
                        dp[kb][nb][i] = see ? x * (dp[kb][nb][i] - dl[i]) * a.scale : 0.0f;
                    }
            }
            accumulate<T, DP, NB>(sgo, p, dv);
            accumulate<T, DP, NB>(sqr, dp, dk);
            }
            };
            if (is_edge(t))
                work_on(std::true_type{});
            else
                work_on(std::false_type{});
            if (threadIdx.x == 0) flags[after == 2 ? 0 : after + 1] = 0;
            turn = after;
            if (kBuffers == 2) {
                buffer ^= 1;
                __syncthreads();
            }
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int key = w0 + 16 * nb + c;
            if (key < a.sinks && key < len) {
                float* out = parts + key * dim;
#pragma unroll
                for (int b = 0; b < DP / 16; ++b) {
                    store_quad(out, 16 * b + 4 * g, dim, dk[b][nb], true);
                    store_quad(out + (int64_t)a.sinks * dim, 16 * b + 4 * g, dim, dv[b][nb], true);
                }
            } else if (!SINKS && key < len) {
                const int64_t at = ((row_base + key) * a.kv_heads + hk) * dim;
#pragma unroll
                for (int b = 0; b < DP / 16; ++b) {
                    store_quad(a.dk + at, 16 * b + 4 * g, dim, dk[b][nb], BUF);
                    store_quad(a.dv + at, 16 * b + 4 * g, dim, dv[b][nb], BUF);
                }
            }
        }
        if (met) {
            __syncthreads();
            const int n = (keys - j0 < kKeys ? keys - j0 : kKeys) * dim;
            for (int e = threadIdx.x; e < n; e += NT) {
                const int key = j0 + e / dim, d = e % dim;
                const int64_t lo = SINKS ? (i0 > key + a.window ? i0 : key + a.window) : key, hi = SINKS ? i1 : (int64_t)key + a.window;
                float x = 0.0f;
                for (int h = h0; h < h0 + heads; ++h)
                    x += not_finite_sum(head_ptr(a.go, a.seq, s, first, h) + d, a.go.st, lo, hi < i1 ? hi : i1);
                if (x == 0.0f) continue;
                if (key < a.sinks)
                    parts[((int64_t)a.sinks + key) * dim + d] += x;
                else
                    a.dv[((row_base + key) * a.kv_heads + hk) * dim + d] = (T)((float)a.dv[((row_base + key) * a.kv_heads + hk) * dim + d] + x);
            }
            met = false;
        }
    }
}

// dK and dV of the sink keys: their window's sums and those of all segments, in order.
template <typename T>
__global__ __launch_bounds__(kThreads) void window_join_kernel(WindowArgs<T> a) {
    const int hk = blockIdx.y, s = blockIdx.z;
    int64_t first, len;
    sequence_rows(a.seq, s, first, len);
    const int64_t n = (int64_t)a.sinks * a.dim, e = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (e >= 2 * n) return;
    const int which = e >= n, key = (int)((e % n) / a.dim), d = (int)(e % a.dim);
    if (key >= len) return;
    const float* p = a.parts + ((int64_t)s * a.kv_heads + hk) * (1 + a.segments) * 2 * n + e;
    float x = 0.0f;
    for (int i = 0; i <= a.segments; i += 16) {
        float part[16];                                        // asked for together, added in order
#pragma unroll
        for (int u = 0; u < 16; ++u) part[u] = i + u <= a.segments ? p[(int64_t)(i + u) * 2 * n] : 0.0f;
#pragma unroll
        for (int u = 0; u < 16; ++u) x += part[u];
    }
    const int64_t row = (a.seq.starts ? first : (int64_t)s * a.seq.max_len) + key;
    (which ? a.dv : a.dk)[(row * a.kv_heads + hk) * a.dim + d] = (T)x;
}

// ---- one row against a rolling cache ----
//
// Slot j < sinks holds row j, slot sinks + r the latest row i >= sinks with (i - sinks) % window == r: exactly the rows
// that row pos[b] sees.  The step stores its own key and value and reads min(pos + 1, sinks + window) slots.

template <typename T>
struct StepArgs {
    Heads<const T> q, k, v;         // (batch, head) rows; st unused
    Heads<T> ck, cv;                // (batch, slot, head)
    const int64_t* pos;
    T* o;
    float* parts;                   // (batch, head, split): maximum, sum, dim values
    int heads, kv_heads, dim, window, sinks, splits, chunks;
    float scale;
    bool whole;                     // rows of k, v and the caches are whole words at 4-byte boundaries
};

// A wave takes kUnroll times 64 / (lanes of a row) consecutive slots at a time; a lane keeps 16 bytes of the row for each of
// GB query heads.  BUF: rows are whole words at 4-byte boundaries (a.whole).
template <typename T, int DP, int GB, bool BUF>
__global__ __launch_bounds__(kThreads) void window_step_kernel(StepArgs<T> a) {
    constexpr int VE = Elem<T>::kPer16B, kLanes = DP / VE, kRows = 64 / kLanes, kUnroll = 4, kTake = kRows * kUnroll;
    static_assert(kTake <= 64, "row_buffer covers 64 rows");
    __shared__ float s_ml[kThreads / 64][GB][2];
    __shared__ float s_acc[kThreads / 64][GB][DP];
    const int split = blockIdx.x, hk = blockIdx.y / a.chunks, chunk = blockIdx.y % a.chunks, b = blockIdx.z;
    const int group = a.heads / a.kv_heads;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), d = lane % kLanes * VE, r = lane / kLanes;
    const int64_t pos = a.pos[b];
    const int slots = a.sinks + a.window;
    const int n = pos < 0 ? 0 : (int)(pos < slots ? pos + 1 : slots);
    const int own = pos < 0 ? -1 : (int)(pos < a.sinks ? pos : a.sinks + (pos - a.sinks) % a.window);
    const int per = (n + a.splits - 1) / a.splits;
    const int lo = split * per, hi = lo + per < n ? lo + per : n;
    T* ck = a.ck.p + b * a.ck.sb + hk * a.ck.sh;
    T* cv = a.cv.p + b * a.cv.sb + hk * a.cv.sh;
    const float l2scale = a.scale * kLog2e;
    // the new row takes its slot's place here, whatever the slot holds: no block waits for the one that stores it
    const u32x4 new_k = load_piece(a.k.p + b * a.k.sb + hk * a.k.sh, d, a.dim, BUF), new_v = load_piece(a.v.p + b * a.v.sb + hk * a.v.sh, d, a.dim, BUF);
    float q[GB][VE], acc[GB][VE], m[GB], sum[GB];
#pragma unroll
    for (int x = 0; x < GB; ++x) {
        const int h = hk * group + chunk * GB + x;
        const bool live = chunk * GB + x < group;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            q[x][e] = live && d + e < a.dim ? (float)a.q.p[b * a.q.sb + h * a.q.sh + d + e] * l2scale : 0.0f;
            acc[x][e] = 0.0f;
        }
        m[x] = -INFINITY;
        sum[x] = 0.0f;
    }
    const int words = (a.dim - d) * (int)sizeof(T) / 4;              // of this lane's piece that are the row's
    for (int base = lo + wave * kTake; base < hi; base += kThreads / 64 * kTake) {
        u32x4 kr[kUnroll], vr[kUnroll];
        if constexpr (BUF) {
            const auto kb = row_buffer(ck + (int64_t)base * a.ck.st, a.ck.st, hi - base < kTake ? hi - base : kTake, a.dim);
            const auto vb = row_buffer(cv + (int64_t)base * a.cv.st, a.cv.st, hi - base < kTake ? hi - base : kTake, a.dim);
            const int col = d < a.dim ? d * (int)sizeof(T) : 1 << 30;
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) kr[u] = load_piece(kb, (u * kRows + r) * (int)a.ck.st * (int)sizeof(T) + col);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) vr[u] = load_piece(vb, (u * kRows + r) * (int)a.cv.st * (int)sizeof(T) + col);
            if (a.dim < DP) {
#pragma unroll
                for (int u = 0; u < kUnroll; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        kr[u][i] = i < words ? kr[u][i] : 0u;
                        vr[u][i] = i < words ? vr[u][i] : 0u;
                    }
            }
        } else {
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const int64_t slot = base + u * kRows + r;
                kr[u] = vr[u] = u32x4{0, 0, 0, 0};
                if (slot < hi) {
                    kr[u] = load_piece(ck + slot * a.ck.st, d, a.dim, false);
                    vr[u] = load_piece(cv + slot * a.cv.st, d, a.dim, false);
                }
            }
        }
        // (slots from hi on are the next split's: a weight of zero would still make NaN of an infinity)
        if (own >= base && own < base + kTake && own < hi) {
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
                if (base + u * kRows + r == own) {
                    kr[u] = new_k;
                    vr[u] = new_v;
                    if (chunk == 0) {
                        store_piece(ck + (int64_t)own * a.ck.st, d, a.dim, new_k, BUF);
                        store_piece(cv + (int64_t)own * a.cv.st, d, a.dim, new_v, BUF);
                    }
                }
        }
        float sc[kUnroll][GB];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            T kk[VE];
            __builtin_memcpy(kk, &kr[u], 16);
            const bool live = base + u * kRows + r < hi;
#pragma unroll
            for (int x = 0; x < GB; ++x) {
                float t = 0.0f;
#pragma unroll
                for (int e = 0; e < VE; ++e) t = fmaf(q[x][e], (float)kk[e], t);
                sc[u][x] = live ? lanes_sum(t, kLanes) : -INFINITY;
            }
        }
#pragma unroll
        for (int x = 0; x < GB; ++x) {
            float now = m[x];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) now = fmaxf(now, sc[u][x]);
            const float ref = now == -INFINITY ? 0.0f : now;
            const float shrink = __builtin_amdgcn_exp2f(m[x] - ref);
            m[x] = now;
            sum[x] *= shrink;
#pragma unroll
            for (int e = 0; e < VE; ++e) acc[x][e] *= shrink;
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                T vv[VE];
                __builtin_memcpy(vv, &vr[u], 16);
                const float p = __builtin_amdgcn_exp2f(sc[u][x] - ref);
                sum[x] += p;
#pragma unroll
                for (int e = 0; e < VE; ++e) acc[x][e] = fmaf(p, (float)vv[e], acc[x][e]);
            }
        }
    }
    // join the rows of a wave, then the waves
#pragma unroll
    for (int x = 0; x < GB; ++x) {
#pragma unroll
        for (int o = kLanes; o < 64; o <<= 1) {
            const float om = __shfl_xor(m[x], o), now = fmaxf(m[x], om), ref = now == -INFINITY ? 0.0f : now;
            const float f = __builtin_amdgcn_exp2f(m[x] - ref), fo = __builtin_amdgcn_exp2f(om - ref);
            sum[x] = sum[x] * f + __shfl_xor(sum[x], o) * fo;
#pragma unroll
            for (int e = 0; e < VE; ++e) acc[x][e] = acc[x][e] * f + __shfl_xor(acc[x][e], o) * fo;
            m[x] = now;
        }
        if (r == 0) {
#pragma unroll
            for (int e = 0; e < VE; ++e) s_acc[wave][x][d + e] = acc[x][e];
            if (d == 0) {
                s_ml[wave][x][0] = m[x];
                s_ml[wave][x][1] = sum[x];
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < GB * DP; i += kThreads) {
        const int x = i / DP, dd = i % DP;
        if (chunk * GB + x >= group || dd >= a.dim) continue;
        float now = -INFINITY, total = 0.0f, value = 0.0f;
#pragma unroll
        for (int w = 0; w < kThreads / 64; ++w) now = fmaxf(now, s_ml[w][x][0]);
        const float ref = now == -INFINITY ? 0.0f : now;
#pragma unroll
        for (int w = 0; w < kThreads / 64; ++w) {
            const float f = __builtin_amdgcn_exp2f(s_ml[w][x][0] - ref);
            total = fmaf(s_ml[w][x][1], f, total);
            value = fmaf(s_acc[w][x][dd], f, value);
        }
        const int64_t head = (int64_t)b * a.heads + hk * group + chunk * GB + x;
        if (a.splits == 1) {
            a.o[head * a.dim + dd] = (T)(n ? value / total : 0.0f);
        } else {
            float* out = a.parts + (head * a.splits + split) * (a.dim + 2);
            out[2 + dd] = value;
            if (dd == 0) {
                out[0] = now;
                out[1] = total;
            }
        }
    }
}

template <typename T>
__global__ __launch_bounds__(128) void window_step_join_kernel(StepArgs<T> a) {
    const int64_t head = blockIdx.x;
    const int d = threadIdx.x;
    if (d >= a.dim) return;
    const float* p = a.parts + head * a.splits * (a.dim + 2);
    const int stride = a.dim + 2;
    float now = -INFINITY, total = 0.0f, value = 0.0f;
#pragma unroll 8
    for (int i = 0; i < a.splits; ++i) now = fmaxf(now, p[i * stride]);
    const float ref = now == -INFINITY ? 0.0f : now;
#pragma unroll 8
    for (int i = 0; i < a.splits; ++i) {
        const float f = __builtin_amdgcn_exp2f(p[i * stride] - ref);
        total = fmaf(p[i * stride + 1], f, total);
        value = fmaf(p[i * stride + 2 + d], f, value);
    }
    a.o[head * a.dim + d] = (T)(a.pos[head / a.heads] < 0 ? 0.0f : value / total);
}

// Rows of whole sequences into their slots: slot by slot, the row that it holds behind the sequence's last.
template <typename T>
__global__ __launch_bounds__(kThreads) void window_fill_kernel(StepArgs<T> a, Sequences seq, int64_t* __restrict__ pos) {
    const int hk = blockIdx.y, b = blockIdx.z;
    int64_t first, len;
    sequence_rows(seq, b, first, len);
    if (pos && blockIdx.x == 0 && hk == 0 && threadIdx.x == 0) pos[b] = len;
    const T* kp = head_ptr(a.k, seq, b, first, hk);
    const T* vp = head_ptr(a.v, seq, b, first, hk);
    T* ck = a.ck.p + b * a.ck.sb + hk * a.ck.sh;
    T* cv = a.cv.p + b * a.cv.sb + hk * a.cv.sh;
    const int pieces = (a.dim + Elem<T>::kPer16B - 1) / Elem<T>::kPer16B;
    const int64_t total = (int64_t)(a.sinks + a.window) * pieces;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
        const int64_t slot = i / pieces;
        const int d = (int)(i % pieces) * Elem<T>::kPer16B;
        int64_t row = slot;
        if (slot >= a.sinks) {
            const int64_t rolled = len - a.sinks, at = slot - a.sinks;
            row = at < rolled ? a.sinks + at + (rolled - 1 - at) / a.window * a.window : len;
        }
        if (row >= len) continue;
        store_piece(ck + slot * a.ck.st, d, a.dim, load_piece(kp + row * a.k.st, d, a.dim, a.whole), a.whole);
        store_piece(cv + slot * a.cv.st, d, a.dim, load_piece(vp + row * a.v.st, d, a.dim, a.whole), a.whole);
    }
}

template <typename T>
Heads<const T> heads_of(const void* p, const int64_t* s) {
    return {static_cast<const T*>(p), s[0], s[1], s[2]};
}

constexpr int64_t kMostBlocks = ((int64_t)1 << 32) / kThreads - 1;

template <typename F>
void for_dim(int dim, F f) {
    if (dim <= 32)
        f(std::integral_constant<int, 32>{});
    else if (dim <= 64)
        f(std::integral_constant<int, 64>{});
    else
        f(std::integral_constant<int, 128>{});
}

// Blocks per head and sequence: one per tile of own rows, fewer (each then takes several) where a launch, whose threads are
// counted in 32 bits, could not hold them.
unsigned row_tiles(int64_t max_len, int rows, int64_t heads) {
    const int64_t n = (max_len + rows - 1) / rows, most = kMostBlocks / heads;
    return (unsigned)(n < 1 ? 1 : (n < most ? n : most));
}

template <typename T, int DP, bool BUF>
struct Kernels {
    // 16-row blocks of own rows per wave.  Two read a streamed tile half as often, one makes twice the blocks and leaves registers
    // for more waves.  O takes two where they still make two rounds of blocks and the window's middle outweighs its edges, and at 128
    // columns always: 4 sequences (2 of 128 columns) of 8192 rows, 16 heads, window 1000: 270 us with two and 315 with one at 64 columns,
    // 172 and 186 at 32, 223 and 268 at 128; a single one 82 and 82; 8 sequences of up to 2000 rows, 8 heads, window 300: 47 and 41 us; 32
    // of up to 1000 rows, 16 heads, window 100: 95 and 91.  dQ (503 and 456 us at 64 columns), dK and dV (528
    // and 527; 100 and 68 on the short ones) take one: at 128 columns two do not fit the registers.
    static constexpr int NK = 1;
    static constexpr size_t kLds = TileShape<T, DP>::lds(TileShape<T, DP>::kBuffers), kLdsSinks = TileShape<T, DP>::lds(1);
    static bool two_blocks(const WindowArgs<T>& a) {
        const int64_t dense = (int64_t)a.n_seq * a.seq.max_len, rows = a.seq.starts && a.seq.n_tokens < dense ? a.seq.n_tokens : dense;
        return rows / 128 * a.heads >= 2048 && a.window >= 256;
    }
    template <int NB>
    static void rows(WindowArgs<T> a, hipStream_t st) {
        a.tiles = row_tiles(a.seq.max_len, 64 * NB, (int64_t)a.heads * a.n_seq);
        hipLaunchKernelGGL((window_rows_kernel<T, DP, NB, false, BUF>), dim3(a.tiles * a.heads * a.n_seq), dim3(kThreads), kLds, st, a);
    }
    static void forward(const WindowArgs<T>& a, hipStream_t st) {
        if constexpr (sizeof(T) == 4)
            rows<1>(a, st);
        else if constexpr (DP == 128)
            rows<2>(a, st);
        else
            two_blocks(a) ? rows<2>(a, st) : rows<1>(a, st);
    }
    static void backward(WindowArgs<T> a, hipStream_t st) {
        const dim3 block(kThreads);
        a.tiles = row_tiles(a.seq.max_len, 64 * NK, (int64_t)a.heads * a.n_seq);
        hipLaunchKernelGGL((window_rows_kernel<T, DP, NK, true, BUF>), dim3(a.tiles * a.heads * a.n_seq), block, kLds, st, a);
        hipLaunchKernelGGL((window_keys_kernel<T, DP, NK, false, BUF>), dim3(a.tiles * a.kv_heads * a.n_seq), block, kLds, st, a);
        if (a.sinks > 0) {
            a.tiles = a.segments * ((a.sinks + 15) / 16);
            hipLaunchKernelGGL((window_keys_kernel<T, DP, 1, true, BUF>), dim3(a.tiles * a.kv_heads * a.n_seq), dim3(64), kLdsSinks, st, a);
            hipLaunchKernelGGL((window_join_kernel<T>), dim3((2 * a.sinks * a.dim + kThreads - 1) / kThreads, a.kv_heads, a.n_seq), block, 0, st, a);
        }
    }
    static int allow() {
        constexpr int kOne = sizeof(T) == 2 && DP == 128 ? 2 : 1, kTwo = sizeof(T) == 2 ? 2 : 1;
        const void* f[] = {reinterpret_cast<const void*>(&window_rows_kernel<T, DP, kOne, false, BUF>), reinterpret_cast<const void*>(&window_rows_kernel<T, DP, kTwo, false, BUF>),
                           reinterpret_cast<const void*>(&window_rows_kernel<T, DP, NK, true, BUF>),
                           reinterpret_cast<const void*>(&window_keys_kernel<T, DP, NK, false, BUF>), reinterpret_cast<const void*>(&window_keys_kernel<T, DP, 1, true, BUF>)};
        for (const void* k : f) VAD_HIP_CHECK(hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)kLds));
        return VAD_OK;
    }
};

template <typename T>
int run_forward(const WindowArgs<T>& a, hipStream_t st) {
    for_dim(a.dim, [&](auto dp) {
        constexpr int DP = decltype(dp)::value;
        a.whole ? Kernels<T, DP, true>::forward(a, st) : Kernels<T, DP, false>::forward(a, st);
    });
    VAD_HIP_CHECK(hipGetLastError());
    return VAD_OK;
}

template <typename T>
int run_backward(const WindowArgs<T>& a, hipStream_t st) {
    for_dim(a.dim, [&](auto dp) {
        constexpr int DP = decltype(dp)::value;
        a.whole ? Kernels<T, DP, true>::backward(a, st) : Kernels<T, DP, false>::backward(a, st);
    });
    VAD_HIP_CHECK(hipGetLastError());
    return VAD_OK;
}

template <typename T, int DP>
int allow_tiles() {
    const int rc = Kernels<T, DP, true>::allow();
    return rc != VAD_OK ? rc : Kernels<T, DP, false>::allow();
}

// Segments (cuts of the rows beyond the window times query heads of a key head) for the sink keys' gradients: at least one
// tile of rows each, enough one-wave blocks to fill the chip.
int sink_segments(int64_t n_seq, int64_t max_len, int heads, int kv_heads, int window) {
    const int64_t beyond = max_len > window ? max_len - window : 0, blocks = n_seq * heads;
    int64_t n = (2048 + blocks - 1) / blocks;
    if (n > beyond / kTile) n = beyond / kTile;
    return (int)(n < 1 ? 1 : n) * (heads / kv_heads);
}

int check_heads(int64_t n_seq, int64_t n_tokens, int64_t max_len, int heads, int kv_heads, int dim, int dtype, int64_t window, int sinks) {
    VAD_REQUIRE(dtype == VAD_DTYPE_F32 || dtype == VAD_DTYPE_BF16, "dtype must be VAD_DTYPE_F32 or VAD_DTYPE_BF16, got %d", dtype);
    VAD_REQUIRE(dim >= 1 && dim <= VAD_MAX_HEAD_DIM, "head dimension %d out of range 1..%d", dim, VAD_MAX_HEAD_DIM);
    VAD_REQUIRE(kv_heads >= 1 && heads >= 1 && heads % kv_heads == 0 && heads <= 65535, "%d heads cannot share %d key heads", heads, kv_heads);
    VAD_REQUIRE(window >= 1 && window <= (1 << 30), "window %lld out of range", (long long)window);
    VAD_REQUIRE(sinks >= 0 && sinks <= VAD_MAX_SINKS, "sinks %d out of range 0..%d", sinks, VAD_MAX_SINKS);
    VAD_REQUIRE(n_seq >= 0 && n_seq <= 65535, "sequence count %lld out of range 0..65535", (long long)n_seq);
    VAD_REQUIRE(n_tokens >= 0 && max_len >= 0 && n_tokens <= (1 << 30) && max_len <= (1 << 30), "length out of range");
    VAD_REQUIRE(n_seq * heads <= kMostBlocks / 2, "too many sequences for one launch");
    VAD_REQUIRE((int64_t)heads * dim < VAD_MAX_ROW_STRIDE, "rows of %lld elements are too long", (long long)heads * dim);
    return VAD_OK;
}

int check_rows(const int64_t* strides) {
    VAD_REQUIRE(strides[1] >= 0 && strides[1] < VAD_MAX_ROW_STRIDE, "row stride %lld out of range", (long long)strides[1]);
    return VAD_OK;
}

}  // namespace

// The tiles of 33 and more columns of float32, 65 and more of bfloat16, use more than 64 KB of LDS: opt in once per device.
int ensure_window_attention_attrs() {
    static std::mutex mu;
    static bool done[64] = {false};
    int dev = 0;
    VAD_HIP_CHECK(hipGetDevice(&dev));
    VAD_REQUIRE(dev >= 0 && dev < 64, "device index %d out of range", dev);
    std::lock_guard<std::mutex> lock(mu);
    if (done[dev]) return VAD_OK;
    int rc = VAD_OK;
    if ((rc = allow_tiles<float, 32>()) != VAD_OK || (rc = allow_tiles<float, 64>()) != VAD_OK || (rc = allow_tiles<float, 128>()) != VAD_OK ||
        (rc = allow_tiles<__bf16, 32>()) != VAD_OK || (rc = allow_tiles<__bf16, 64>()) != VAD_OK || (rc = allow_tiles<__bf16, 128>()) != VAD_OK)
        return rc;
    done[dev] = true;
    return VAD_OK;
}
}  // namespace vad

extern "C" int vad_window_attention_forward(const void* q_dev, const int64_t* q_strides, const void* k_dev, const int64_t* k_strides,
                                            const void* v_dev, const int64_t* v_strides, const int64_t* starts_dev, int64_t n_seq,
                                            int64_t n_tokens, int64_t max_len, int heads, int kv_heads, int dim, int dtype, int64_t window,
                                            int sinks, float scale, void* o_dev, float* stats_dev, void* stream) {
    using namespace vad;
    int rc = check_heads(n_seq, n_tokens, max_len, heads, kv_heads, dim, dtype, window, sinks);
    if (rc != VAD_OK) return rc;
    VAD_REQUIRE(scale > 0.0f && scale < INFINITY, "scale must be positive and finite");
    VAD_REQUIRE(q_strides && k_strides && v_strides, "null pointer argument");
    if (n_seq == 0 || (starts_dev ? n_tokens : max_len) == 0) return VAD_OK;
    VAD_REQUIRE(q_dev && k_dev && v_dev && o_dev, "null pointer argument");
    for (const int64_t* strides : {q_strides, k_strides, v_strides})
        if ((rc = check_rows(strides)) != VAD_OK) return rc;
    rc = ensure_window_attention_attrs();
    if (rc != VAD_OK) return rc;
    const auto run = [&](auto zero) {
        typedef decltype(zero) T;
        WindowArgs<T> a = {};
        a.q = heads_of<T>(q_dev, q_strides);
        a.k = heads_of<T>(k_dev, k_strides);
        a.v = heads_of<T>(v_dev, v_strides);
        a.out = static_cast<T*>(o_dev);
        a.stats = stats_dev;
        a.seq = {starts_dev, n_tokens, max_len};
        a.n_seq = (int)n_seq, a.heads = heads, a.kv_heads = kv_heads, a.dim = dim;
        a.window = (int)window, a.sinks = sinks, a.scale = scale;
        a.whole = whole_rows(a.q, dim) && whole_rows(a.k, dim) && whole_rows(a.v, dim) && whole_words(a.out, dim);
        return run_forward<T>(a, static_cast<hipStream_t>(stream));
    };
    return dtype == VAD_DTYPE_F32 ? run(0.0f) : run((__bf16)0.0f);
}

extern "C" size_t vad_window_attention_workspace_bytes(int64_t n_seq, int64_t n_rows, int64_t max_len, int heads, int kv_heads, int dim,
                                                       int64_t window, int sinks) {
    using namespace vad;
    if (n_seq <= 0 || n_rows <= 0 || heads <= 0 || kv_heads <= 0 || dim <= 0 || window <= 0 || sinks < 0) return 0;
    size_t floats = (size_t)n_rows * heads;
    if (sinks > 0) floats += (size_t)n_seq * kv_heads * (1 + sink_segments(n_seq, max_len, heads, kv_heads, (int)window)) * 2 * sinks * dim;
    return floats * sizeof(float);
}

extern "C" int vad_window_attention_backward(const void* q_dev, const int64_t* q_strides, const void* k_dev, const int64_t* k_strides,
                                             const void* v_dev, const int64_t* v_strides, const void* o_dev, const void* do_dev,
                                             const int64_t* do_strides, const float* stats_dev, const int64_t* starts_dev, int64_t n_seq,
                                             int64_t n_tokens, int64_t max_len, int heads, int kv_heads, int dim, int dtype,
                                             int64_t window, int sinks, float scale, void* dq_dev, void* dk_dev, void* dv_dev,
                                             void* workspace_dev, size_t workspace_bytes, void* stream) {
    using namespace vad;
    int rc = check_heads(n_seq, n_tokens, max_len, heads, kv_heads, dim, dtype, window, sinks);
    if (rc != VAD_OK) return rc;
    VAD_REQUIRE(scale > 0.0f && scale < INFINITY, "scale must be positive and finite");
    VAD_REQUIRE(q_strides && k_strides && v_strides && do_strides, "null pointer argument");
    if (n_seq == 0 || (starts_dev ? n_tokens : max_len) == 0) return VAD_OK;
    VAD_REQUIRE(q_dev && k_dev && v_dev && o_dev && do_dev && stats_dev && dq_dev && dk_dev && dv_dev && workspace_dev, "null pointer argument");
    for (const int64_t* strides : {q_strides, k_strides, v_strides, do_strides})
        if ((rc = check_rows(strides)) != VAD_OK) return rc;
    const int64_t n_rows = starts_dev ? n_tokens : n_seq * max_len;
    const size_t need = vad_window_attention_workspace_bytes(n_seq, n_rows, max_len, heads, kv_heads, dim, window, sinks);
    VAD_REQUIRE(workspace_bytes >= need, "workspace of %zu bytes is too small: %zu", workspace_bytes, need);
    rc = ensure_window_attention_attrs();
    if (rc != VAD_OK) return rc;
    const auto run = [&](auto zero) {
        typedef decltype(zero) T;
        WindowArgs<T> a = {};
        a.q = heads_of<T>(q_dev, q_strides);
        a.k = heads_of<T>(k_dev, k_strides);
        a.v = heads_of<T>(v_dev, v_strides);
        a.go = heads_of<T>(do_dev, do_strides);
        a.o = static_cast<const T*>(o_dev);
        a.out = static_cast<T*>(dq_dev);
        a.dk = static_cast<T*>(dk_dev);
        a.dv = static_cast<T*>(dv_dev);
        a.stats = const_cast<float*>(stats_dev);
        a.delta = static_cast<float*>(workspace_dev);
        a.parts = a.delta + n_rows * heads;
        a.seq = {starts_dev, n_tokens, max_len};
        a.n_seq = (int)n_seq, a.heads = heads, a.kv_heads = kv_heads, a.dim = dim;
        a.window = (int)window, a.sinks = sinks, a.scale = scale;
        a.segments = sink_segments(n_seq, max_len, heads, kv_heads, (int)window);
        a.whole = whole_rows(a.q, dim) && whole_rows(a.k, dim) && whole_rows(a.v, dim) && whole_rows(a.go, dim) && whole_words(a.o, dim) &&
                  whole_words(a.out, dim) && whole_words(a.dk, dim) && whole_words(a.dv, dim);
        return run_backward<T>(a, static_cast<hipStream_t>(stream));
    };
    return dtype == VAD_DTYPE_F32 ? run(0.0f) : run((__bf16)0.0f);
}

namespace vad {
namespace {

// Splits of a row's slots: enough blocks to fill the chip, at least 64 slots each.
int step_splits(int64_t batch, int kv_heads, int chunks, int64_t slots) {
    const int64_t blocks = batch * kv_heads * chunks;
    int64_t n = (1024 + blocks - 1) / blocks;
    if (n > slots / 64) n = slots / 64;
    if (n > 64) n = 64;
    return (int)(n < 1 ? 1 : n);
}
int step_heads(int group) { return group >= 4 ? 4 : (group >= 2 ? 2 : 1); }      // query heads of a block

template <typename T>
int run_step(StepArgs<T> a, int64_t batch, hipStream_t st) {
    const int group = a.heads / a.kv_heads, gb = step_heads(group);
    const dim3 grid(a.splits, a.kv_heads * a.chunks, (unsigned)batch), block(kThreads);
    for_dim(a.dim, [&](auto dp) {
        constexpr int DP = decltype(dp)::value;
        const auto launch = [&](auto heads) {
            constexpr int GB = decltype(heads)::value;
            if (a.whole)
                hipLaunchKernelGGL((window_step_kernel<T, DP, GB, true>), grid, block, 0, st, a);
            else
                hipLaunchKernelGGL((window_step_kernel<T, DP, GB, false>), grid, block, 0, st, a);
        };
        if (gb == 4)
            launch(std::integral_constant<int, 4>{});
        else if (gb == 2)
            launch(std::integral_constant<int, 2>{});
        else
            launch(std::integral_constant<int, 1>{});
    });
    VAD_HIP_CHECK(hipGetLastError());
    if (a.splits > 1) {
        hipLaunchKernelGGL((window_step_join_kernel<T>), dim3((unsigned)(batch * a.heads)), dim3(128), 0, st, a);
        VAD_HIP_CHECK(hipGetLastError());
    }
    return VAD_OK;
}

}  // namespace
}  // namespace vad

extern "C" size_t vad_window_step_workspace_bytes(int64_t batch, int heads, int kv_heads, int dim, int64_t window, int sinks) {
    using namespace vad;
    if (batch <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || dim <= 0 || window <= 0 || sinks < 0) return 0;
    const int group = heads / kv_heads, gb = step_heads(group), splits = step_splits(batch, kv_heads, (group + gb - 1) / gb, sinks + window);
    return splits > 1 ? (size_t)batch * heads * splits * (dim + 2) * sizeof(float) : 0;
}

extern "C" int vad_window_attention_step(const void* q_dev, const int64_t* q_strides, const void* k_dev, const int64_t* k_strides,
                                         const void* v_dev, const int64_t* v_strides, void* cache_k_dev, const int64_t* cache_k_strides,
                                         void* cache_v_dev, const int64_t* cache_v_strides, const int64_t* pos_dev, int64_t batch,
                                         int heads, int kv_heads, int dim, int dtype, int64_t window, int sinks, float scale, void* o_dev,
                                         void* workspace_dev, size_t workspace_bytes, void* stream) {
    using namespace vad;
    int rc = check_heads(batch, 0, 0, heads, kv_heads, dim, dtype, window, sinks);
    if (rc != VAD_OK) return rc;
    VAD_REQUIRE(scale > 0.0f && scale < INFINITY, "scale must be positive and finite");
    if (batch == 0) return VAD_OK;
    VAD_REQUIRE(q_dev && k_dev && v_dev && cache_k_dev && cache_v_dev && pos_dev && o_dev && q_strides && k_strides && v_strides &&
                    cache_k_strides && cache_v_strides,
                "null pointer argument");
    const size_t need = vad_window_step_workspace_bytes(batch, heads, kv_heads, dim, window, sinks);
    VAD_REQUIRE(workspace_bytes >= need && (!need || workspace_dev), "workspace of %zu bytes is too small: %zu", workspace_bytes, need);
    const auto run = [&](auto zero) {
        typedef decltype(zero) T;
        StepArgs<T> a = {};
        a.q = {static_cast<const T*>(q_dev), q_strides[0], 0, q_strides[1]};
        a.k = {static_cast<const T*>(k_dev), k_strides[0], 0, k_strides[1]};
        a.v = {static_cast<const T*>(v_dev), v_strides[0], 0, v_strides[1]};
        a.ck = {static_cast<T*>(cache_k_dev), cache_k_strides[0], cache_k_strides[1], cache_k_strides[2]};
        a.cv = {static_cast<T*>(cache_v_dev), cache_v_strides[0], cache_v_strides[1], cache_v_strides[2]};
        a.pos = pos_dev;
        a.o = static_cast<T*>(o_dev);
        a.parts = static_cast<float*>(workspace_dev);
        a.heads = heads, a.kv_heads = kv_heads, a.dim = dim, a.window = (int)window, a.sinks = sinks, a.scale = scale;
        const int group = heads / kv_heads, gb = step_heads(group);
        a.chunks = (group + gb - 1) / gb;
        a.splits = step_splits(batch, kv_heads, a.chunks, sinks + window);
        // A cache may be laid out with any slot stride.  A buffer takes those below VAD_MAX_ROW_STRIDE, and ends with the last slot
        // only where slots lie behind one another: that of a single slot may be anything.
        a.whole = whole_words(a.k, dim) && whole_words(a.v, dim) && whole_words(a.ck, dim) && whole_words(a.cv, dim);
        for (const int64_t st : {a.ck.st, a.cv.st}) a.whole = a.whole && st >= dim && st < VAD_MAX_ROW_STRIDE;
        return run_step<T>(a, batch, static_cast<hipStream_t>(stream));
    };
    return dtype == VAD_DTYPE_F32 ? run(0.0f) : run((__bf16)0.0f);
}

extern "C" int vad_window_cache_fill(const void* k_dev, const int64_t* k_strides, const void* v_dev, const int64_t* v_strides,
                                     const int64_t* starts_dev, int64_t n_seq, int64_t n_tokens, int64_t max_len, int kv_heads, int dim,
                                     int dtype, int64_t window, int sinks, void* cache_k_dev, const int64_t* cache_k_strides,
                                     void* cache_v_dev, const int64_t* cache_v_strides, int64_t* pos_dev, void* stream) {
    using namespace vad;
    int rc = check_heads(n_seq, n_tokens, max_len, kv_heads, kv_heads, dim, dtype, window, sinks);
    if (rc != VAD_OK) return rc;
    if (n_seq == 0) return VAD_OK;
    const bool empty = (starts_dev ? n_tokens : max_len) == 0;
    VAD_REQUIRE(k_strides && v_strides && cache_k_strides && cache_v_strides && cache_k_dev && cache_v_dev && (empty || (k_dev && v_dev)),
                "null pointer argument");
    const auto run = [&](auto zero) {
        typedef decltype(zero) T;
        StepArgs<T> a = {};
        a.k = heads_of<T>(k_dev, k_strides);
        a.v = heads_of<T>(v_dev, v_strides);
        a.ck = {static_cast<T*>(cache_k_dev), cache_k_strides[0], cache_k_strides[1], cache_k_strides[2]};
        a.cv = {static_cast<T*>(cache_v_dev), cache_v_strides[0], cache_v_strides[1], cache_v_strides[2]};
        a.kv_heads = kv_heads, a.dim = dim, a.window = (int)window, a.sinks = sinks;
        a.whole = whole_words(a.k, dim) && whole_words(a.v, dim) && whole_words(a.ck, dim) && whole_words(a.cv, dim);
        const Sequences seq = {starts_dev, n_tokens, max_len};
        const int64_t blocks = (((int64_t)sinks + window) * dim * sizeof(T) / 16 + kThreads) / kThreads;
        hipLaunchKernelGGL((window_fill_kernel<T>), dim3((unsigned)(blocks < 256 ? blocks : 256), kv_heads, (unsigned)n_seq), dim3(kThreads), 0,
                           static_cast<hipStream_t>(stream), a, seq, pos_dev);
        VAD_HIP_CHECK(hipGetLastError());
        return (int)VAD_OK;
    };
    return dtype == VAD_DTYPE_F32 ? run(0.0f) : run((__bf16)0.0f);
}
