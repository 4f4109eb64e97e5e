// Linear attention with a decay per head: the recurrent layer S_t = a S_{t-1} + k_t v_t^T, o_t = s q_t S_t with
// a = exp(log_decay[head]), over whole sequences in pieces of 64 rows, its backward pass, and one step of it.
//
// Within a piece (rows i, j counted from its first row) with H = a S, S the state behind the row before it,
//   o_i = s a^i q_i H + s sum_{j <= i} a^(i-j) (q_i . k_j) v_j,      H' = a^n H + sum_j a^(n-j) k_j v_j^T
// so a piece is four small matrix products and the state crosses from piece to piece in the registers of the block
// that walks along a sequence and head.  The backward pass is the same walk three times over:
//   dq: (q,k,v) = (do, v, k) forwards, with S transposed;  dk: (v, do, q) backwards;  dv: (k, q, do) backwards
// the backward walks starting from the gradient of the final state and ending at a times that of the initial state.
//
// Where sequences and heads alone do not fill the chip, a sequence is cut into spans walked by blocks of their own: a
// first launch computes each span's state from k and v alone, and the walk of every span starts from those before it --
// added up by its block, or, where the spans are many, by a launch in between that goes along the sequence once.
//
// Measured, bfloat16 heads of 64: 4 x 16 heads of 8192 rows in 99 us (states of the spans 27, their join 6, walk 65: 268 MB
// at 2.7 TB/s, where a copy takes 57 us -- latency along a walk and vector work on its 64 x 64 weights bound it, not memory);
// 24 ragged sequences of up to 2000 rows and 8 heads, with gradients, 189 us.  A step of 64 x 16 states of 128 x 128 22.9 us:
// 134 MB read and written, 5.9 TB/s with what the last cache keeps.  (Passes in a row; the comparisons beside the choices below
// were taken in turn on a card that had just been idle, where the same kernels are up to a tenth slower.)
//
// Wave w of a block owns columns 16 w .. 16 w + 15 of the state and of the outputs.  The state stays in float32; for
// bfloat16 inputs its update multiplies v by the decay in float32 and splits the product into bfloat16 terms -- three, which
// is exact, where the state is handed out or crosses spans, two (2^-17) where it only feeds outputs of 8 bits.  The weights
// a^(i-j) (q . k) and the copy of the state that q is multiplied with are rounded to bfloat16 once.

#include <mutex>

#include "sequence_device.h"

namespace vad {
namespace {
using namespace sq;

constexpr int kPiece = 64;

template <typename T>
struct Walk {
    Heads<const T> q, k, v;
    T* o;                              // rows of heads * dim
    const float* s0;                   // initial state (n_seq, heads, dim, dim) or null
    float* s1;                         // final state or null
    float within, across, update;      // factors of the piece's own products, of q H, and of k v^T
    bool s0_transposed, reverse;
};

template <typename T>
struct WalkArgs {
    Walk<T> walk[3];
    Sequences seq;
    const float* log_decay;
    float* spans;                      // [walk][seq][head][span][dim][dim]
    int n_seq, heads, dim, n_spans;
    bool joined;                       // spans hold the states that they start from, not those that they leave
    bool whole;                        // all rows are whole words at 4-byte boundaries
};

__device__ __forceinline__ float log2_decay(float ld) {
    // not validated on the host (it lives on the device): a growing state or one past float32 is cut off, NaN stays
    ld = ld > 0.0f ? 0.0f : (ld < -87.0f ? -87.0f : ld);
    return ld * kLog2e;
}
__device__ __forceinline__ float power(float l2, float n) { return __builtin_amdgcn_exp2f(l2 * n); }

// rows of a span: sequences shorter than the hint are cut just as evenly
__device__ __forceinline__ int64_t span_rows(int64_t len, int n_spans) {
    const int64_t per = (len + n_spans - 1) / n_spans;
    return per <= kPiece ? kPiece : (per + kPiece - 1) / kPiece * kPiece;
}

template <typename T, int DP>
struct WalkShape {
    static constexpr int kWaves = DP / 16;
    static constexpr int kThreads = kWaves * 64;
    static constexpr int kLd = DP + Elem<T>::kPer16B;
    static constexpr int kLdP = kPiece + Elem<T>::kPer16B;
    static constexpr size_t kLds = (size_t)(3 * kPiece * kLd + kPiece * kLdP) * sizeof(T) + 16;
};

// The (row block, key block) pairs of a piece's weights: the lower triangle, and the two blocks above it that share a
// contraction of 32 keys with a diagonal block and must read as zero.  Two bits a pair.
constexpr unsigned pack_pairs(int which) {
    const int p[12][2] = {{0, 0}, {1, 0}, {1, 1}, {2, 0}, {2, 1}, {2, 2}, {3, 0}, {3, 1}, {3, 2}, {3, 3}, {0, 1}, {2, 3}};
    unsigned r = 0;
    for (int t = 0; t < 12; ++t) r |= (unsigned)p[t][which] << (2 * t);
    return r;
}

// float32 values as the sum of three bfloat16 (24 bits); not-finite values in the first term alone
__device__ __forceinline__ void split3(const float (&x)[8], bf16x8 (&f)[3]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const __bf16 hi = (__bf16)x[j];
        const float r = fabsf(x[j]) < INFINITY ? x[j] - (float)hi : 0.0f;
        const __bf16 mid = (__bf16)r;
        f[0][j] = hi;
        f[1][j] = mid;
        f[2][j] = (__bf16)(r - (float)mid);
    }
}

// Waves per SIMD that the registers are shared out for.
template <typename T, int DP, bool STATE>
constexpr int walk_waves() { return sizeof(T) == 2 && STATE ? 4 : (sizeof(T) == 2 && DP < 128 ? 3 : 2); }

// BUF: rows are whole words at 4-byte boundaries (a.whole).
template <typename T, int DP, bool STATE, bool BUF>
__global__ __launch_bounds__(DP * 4, (walk_waves<T, DP, STATE>())) void decay_walk_kernel(WalkArgs<T> a) {
    using C = WalkShape<T, DP>;
    extern __shared__ char lds_raw[];
    T* sk = reinterpret_cast<T*>(lds_raw);
    T* sv = sk + kPiece * C::kLd;
    T* sq_ = sv + kPiece * C::kLd;
    T* sp = sq_ + kPiece * C::kLd;
    int* flags = reinterpret_cast<int*>(sp + kPiece * C::kLdP);

    const int h = blockIdx.x % a.heads;
    const int span = (blockIdx.x / a.heads) % a.n_spans;
    const int s = blockIdx.x / a.heads / a.n_spans;
    const Walk<T> w = a.walk[blockIdx.y];
    int64_t first, len;
    sequence_rows(a.seq, s, first, len);
    const int dim = a.dim;
    if (!STATE) zero_outside(w.o, (int64_t)a.heads * dim, h * dim, dim, a.seq, s, a.n_seq, span, a.n_spans);
    const int64_t per = span_rows(len, a.n_spans);
    const int64_t t0 = span * per, t1 = t0 + per < len ? t0 + per : len;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    const int64_t head = (int64_t)s * a.heads + h, elems = (int64_t)dim * dim;
    float* spans = a.spans ? a.spans + (((int64_t)blockIdx.y * a.n_seq * a.heads + head) * a.n_spans + span) * elems : nullptr;
    if (STATE) {
        if (t0 >= len || t1 == len) return;        // the last span's own state is not needed
    } else if (len == 0 && span == 0) {
        if (w.s1)
            for (int64_t i = threadIdx.x; i < elems; i += C::kThreads) w.s1[head * elems + i] = w.s0 ? w.s0[head * elems + i] : 0.0f;
        return;
    } else if (t0 >= len) {
        return;
    }
    const float l2 = log2_decay(a.log_decay[h]);

    // H: block b holds rows 16 b + 4 g + i, column 16 wave + c
    f32x4 H[DP / 16];
    const int col = 16 * wave + c;
#pragma unroll
    for (int b = 0; b < DP / 16; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = 16 * b + 4 * g + i;
            float x = 0.0f;
            if (!STATE && row < dim && col < dim) {
                if (a.joined)
                    x = spans[row * dim + col];
                else if (w.s0)
                    x = w.s0[head * elems + (w.s0_transposed ? col * dim + row : row * dim + col)] * (w.reverse ? 1.0f : power(l2, 1.0f));
            }
            H[b][i] = x;
        }

    if (!STATE && a.n_spans > 1 && !a.joined) {
        const float keep = power(l2, (float)per);
        const float* before = spans - (int64_t)span * elems;
#pragma unroll 1
        for (int u = 0; u < span; ++u, before += elems) {
            f32x4 own[DP / 16];
#pragma unroll
            for (int b = 0; b < DP / 16; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = 16 * b + 4 * g + i;
                    own[b][i] = row < dim && col < dim ? before[row * dim + col] : 0.0f;
                }
#pragma unroll
            for (int b = 0; b < DP / 16; ++b) H[b] = H[b] * keep + own[b];
        }
    }

    const T* kp = head_ptr(w.k, a.seq, s, first, h);
    const T* vp = head_ptr(w.v, a.seq, s, first, h);
    const T* qp = STATE ? nullptr : head_ptr(w.q, a.seq, s, first, h);
    T* op = w.o + ((a.seq.starts ? first : (int64_t)s * a.seq.max_len) * a.heads + h) * dim;
    const int sign = w.reverse ? -1 : 1;
    Staged<T, DP, C::kThreads, BUF, C::kLd> rk, rv, rq;
    const auto fetch = [&](int64_t tc) {
        const int64_t at = w.reverse ? len - 1 - tc : tc;
        const int rows = (int)(t1 - tc < kPiece ? t1 - tc : kPiece);
        rk.fetch(kp, w.k.st, at, rows, dim, w.reverse);
        rv.fetch(vp, w.v.st, at, rows, dim, w.reverse);
        if (!STATE) rq.fetch(qp, w.q.st, at, rows, dim, w.reverse);
    };
    // Powers of the decay.  A row and key block m apart need a^(16 m + c - 4 g - i) = a^(16 m - 15) a^c a^(15 - 4 g - i), a
    // diagonal block its own; the state's update a^(64 - row) = a^(16 m') a a^(15 - 4 g - i).
    const float a1 = power(l2, 1.0f), a16 = power(l2, 16.0f), a32 = a16 * a16, ac = power(l2, (float)c);
    const float within = w.within * ac * a1, across = w.across * ac;
    float tail[4], diagonal[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        tail[i] = power(l2, (float)(15 - 4 * g - i));
        diagonal[i] = c >= 4 * g + i ? w.within * power(l2, (float)(c - 4 * g - i)) : 0.0f;
    }
    const bool third = w.s1 || STATE;        // a state that is handed out or crosses spans keeps float32's accuracy
    if (threadIdx.x < 2) flags[threadIdx.x] = 0;
    fetch(t0);
    __syncthreads();
    int turn = 0;
    for (int64_t tc = t0; tc < t1; tc += kPiece, turn ^= 1) {
        const int n = (int)(t1 - tc < kPiece ? t1 - tc : kPiece);
        rk.put(sk, dim);
        rv.put(sv, dim);
        if (!STATE) {
            rq.put(sq_, dim);
            // (of bfloat16 keys as well: 67 -> 69 us on 4 x 16 heads of 8192 rows)
            if (rv.not_finite() | (sizeof(T) == 2 && rk.not_finite())) flags[turn] = 1;
        }
        __syncthreads();
        const bool careful = !STATE && flags[turn];
        if (threadIdx.x == 0) flags[turn ^ 1] = 0;
        if (tc + kPiece < t1) fetch(tc + kPiece);

        f32x4 o[4];
        if (!STATE) {
            // weights of the piece: rows in columns of the tile, keys 16 kb + 4 g + i down its lanes
#pragma unroll
            for (int u = 0; u < (12 + C::kWaves - 1) / C::kWaves; ++u) {
                const int t = wave + u * C::kWaves;
                if (t >= 12) break;
                const int rb = (pack_pairs(0) >> (2 * t)) & 3, kb = (pack_pairs(1) >> (2 * t)) & 3;
                f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
                if (kb <= rb) {
#pragma unroll
                    for (int d = 0; d < DP; d += 32)
                        acc = mma(frag_natural(sk, C::kLd, 16 * kb, d), frag_natural(sq_, C::kLd, 16 * rb, d), acc);
                    if (kb == rb) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[i] = c >= 4 * g + i ? acc[i] * diagonal[i] : 0.0f;
                    } else {
                        const float f = within * (rb - kb == 1 ? 1.0f : (rb - kb == 2 ? a16 : a32));
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[i] = acc[i] * tail[i] * f;
                    }
                }
                Quad<T> p;
#pragma unroll
                for (int i = 0; i < 4; ++i) p[i] = (T)acc[i];
                *reinterpret_cast<Quad<T>*>(sp + (16 * rb + c) * C::kLdP + 16 * kb + 4 * g) = p;
            }
            // q H, transposed: outputs 16 wave + 4 g + i of row 16 rb + c
            Frag<T> hf[DP / 32];
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) to_frag(H[2 * d], H[2 * d + 1], hf[d]);
#pragma unroll
            for (int rb = 0; rb < 4; ++rb) {
                o[rb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int d = 0; d < DP / 32; ++d) o[rb] = mma(hf[d], frag_split(sq_, C::kLd, 16 * rb, 32 * d), o[rb]);
                o[rb] *= across;
                if (rb & 1) o[rb] *= a16;
                if (rb & 2) o[rb] *= a32;
            }
        }
        Frag<T> vf[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) vf[t] = frag_columns(sv, C::kLd, 32 * t, 16 * wave);

        // the state behind the piece
        const bool last = tc + kPiece >= t1;
        const bool finish = !STATE && last && t1 == len && w.s1, updates = !last || STATE || finish;
        const bool less = finish && !w.reverse;                            // the forward walk hands out S, not a S
        if (updates && !careful) {
            const float keep = n == kPiece && !less ? a32 * a32 : power(l2, (float)(n - (less ? 1 : 0)));
#pragma unroll
            for (int b = 0; b < DP / 16; ++b) H[b] *= keep;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                float x[8];
                if (n == kPiece) {
                    // the varying factor first: a product of constants would be kept in registers across the pieces
                    const float f = w.update * (less ? 1.0f : a1) * (t ? 1.0f : a32);
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = (float)vf[t][j] * tail[j & 3] * (j < 4 ? f * a16 : f);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int row = 32 * t + 4 * g + (j < 4 ? j : 12 + j);
                        x[j] = row < n ? (float)vf[t][j] * (w.update * power(l2, (float)(n - row - (less ? 1 : 0)))) : 0.0f;
                    }
                }
                if constexpr (sizeof(T) == 2) {
                    bf16x8 f[3];
                    split3(x, f);
#pragma unroll
                    for (int b = 0; b < DP / 16; ++b) {
                        const bf16x8 kf = frag_columns(sk, C::kLd, 32 * t, 16 * b);
#pragma unroll
                        for (int m = 2; m >= 0; --m)
                            if (m < 2 || third) H[b] = mma(kf, f[m], H[b]);
                    }
                } else {
                    f32x8 f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) f[j] = x[j];
#pragma unroll
                    for (int b = 0; b < DP / 16; ++b) H[b] = mma(frag_columns(sk, C::kLd, 32 * t, 16 * b), f, H[b]);
                }
            }
        }
        if (!STATE) {
            __syncthreads();
            // Infinities and NaN among the piece's v: only rows behind them may feel them, and 0 * inf is NaN.  They stay out
            // of the matrix product and are added key by key.
            if (careful) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int j = 0; j < 8; ++j) vf[t][j] = fabsf((float)vf[t][j]) < INFINITY ? vf[t][j] : (T)0.0f;
            }
#pragma unroll
            for (int rb = 0; rb < 4; ++rb)
#pragma unroll
                for (int t = 0; t <= rb / 2; ++t) o[rb] = mma(vf[t], frag_split(sp, C::kLdP, 16 * rb, 32 * t), o[rb]);
            if (careful) {
#pragma unroll
                for (int rb = 0; rb < 4; ++rb)
#pragma unroll 1
                    for (int key = 0; key <= 16 * rb + c; ++key)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float x = (float)sv[key * C::kLd + 16 * wave + 4 * g + i];
                            if (!(fabsf(x) < INFINITY)) o[rb][i] = fmaf((float)sp[(16 * rb + c) * C::kLdP + key], x, o[rb][i]);
                        }
            }
            T* oc = op + (w.reverse ? len - 1 - tc : tc) * a.heads * dim;
#pragma unroll
            for (int rb = 0; rb < 4; ++rb) {
                const int row = 16 * rb + c;
                if (row < n) store_quad(oc + sign * row * a.heads * dim, 16 * wave + 4 * g, dim, o[rb], BUF);
            }
        }
        if (careful && updates) {
            // Row by row: the matrix product would also multiply infinities and NaN by what is only there for its shape -- the zeros
            // behind a head's columns, the lower terms of a split value, zero or of the other sign -- and 0 * inf is NaN.
            const float keep = power(l2, (float)(n - (less ? 1 : 0)));
#pragma unroll
            for (int b = 0; b < DP / 16; ++b) H[b] *= keep;
#pragma unroll 1
            for (int row = 0; row < n; ++row) {
                const float x = (float)sv[row * C::kLd + col] * (w.update * power(l2, (float)(n - row - (less ? 1 : 0))));
#pragma unroll
                for (int b = 0; b < DP / 16; ++b) {
                    const Quad<T> y = *reinterpret_cast<const Quad<T>*>(sk + row * C::kLd + 16 * b + 4 * g);
#pragma unroll
                    for (int i = 0; i < 4; ++i) H[b][i] = 16 * b + 4 * g + i < dim ? fmaf((float)y[i], x, H[b][i]) : 0.0f;
                }
            }
        }
        __syncthreads();
    }
    if (STATE && sizeof(T) == 2) {
        // A NaN in a span's state: perhaps an infinity's meeting with a lower term.  Once more, row by row: 1 ms where one
        // of 4 x 8192 rows is NaN, and nothing where none is.
        bool spoilt = false;
#pragma unroll
        for (int b = 0; b < DP / 16; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) spoilt |= H[b][i] != H[b][i];
        if (__any(spoilt)) {
#pragma unroll
            for (int b = 0; b < DP / 16; ++b) H[b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
            for (int64_t t = t0; t < t1 && col < dim; ++t) {
                const int64_t at = w.reverse ? len - 1 - t : t;
                const float x = (float)vp[at * w.v.st + col] * (w.update * power(l2, (float)(t1 - t)));
#pragma unroll
                for (int b = 0; b < DP / 16; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int d = 16 * b + 4 * g + i;
                        if (d < dim) H[b][i] = fmaf((float)kp[at * w.k.st + d], x, H[b][i]);
                    }
            }
        }
    }
    float* out = STATE ? spans : (t1 == len && w.s1 ? w.s1 + head * elems : nullptr);
    if (out) {
#pragma unroll
        for (int b = 0; b < DP / 16; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = 16 * b + 4 * g + i;
                if (row < dim && col < dim) out[row * dim + col] = H[b][i];
            }
    }
}

// spans[u] on entry: the state that span u alone leaves; on return: the state that span u starts from.
template <typename T>
__global__ __launch_bounds__(256) void decay_join_kernel(WalkArgs<T> a) {
    const int64_t elems = (int64_t)a.dim * a.dim, blocks = (elems + 255) / 256;
    const int64_t head = blockIdx.x / blocks, e = blockIdx.x % blocks * 256 + threadIdx.x;
    const int h = head % a.heads, s = head / a.heads;
    const Walk<T> w = a.walk[blockIdx.y];
    int64_t first, len;
    sequence_rows(a.seq, s, first, len);
    if (e >= elems || len == 0) return;
    const int64_t per = span_rows(len, a.n_spans), used = (len + per - 1) / per;
    const float l2 = log2_decay(a.log_decay[h]), keep = power(l2, (float)per);
    float x = 0.0f;
    if (w.s0) x = w.s0[head * elems + (w.s0_transposed ? e % a.dim * a.dim + e / a.dim : e)] * (w.reverse ? 1.0f : power(l2, 1.0f));
    float* p = a.spans + (((int64_t)blockIdx.y * a.n_seq * a.heads + head) * a.n_spans) * elems + e;
    constexpr int kAhead = 8;                                // loads in flight; the sums are a chain
    for (int64_t u = 0; u < used; u += kAhead) {
        float own[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) own[i] = u + i + 1 < used ? p[(u + i) * elems] : 0.0f;
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (u + i < used) {
                p[(u + i) * elems] = x;
                x = fmaf(x, keep, own[i]);
            }
    }
}

// One step: the state is read, updated and written once.  A block owns 32 columns of one state, VE of them per thread,
// the rows dealt to 8 VE groups of threads.
template <typename T, int VE>
__global__ __launch_bounds__(256) void decay_step_kernel(Heads<const T> q, Heads<const T> k, Heads<const T> v, const float* __restrict__ log_decay,
                                                         float scale, int heads, int dim, int slices, float* __restrict__ state, T* __restrict__ o) {
    typedef float vec __attribute__((ext_vector_type(VE == 1 ? 2 : VE)));
    constexpr int kLanes = 32 / VE, kGroups = 256 / kLanes;
    __shared__ float sums[4][32];
    const int64_t head = blockIdx.x / slices;
    const int h = head % heads, b = head / heads;
    const int c = blockIdx.x % slices * 32 + threadIdx.x % kLanes * VE, group = threadIdx.x / kLanes;
    const float a = __builtin_amdgcn_exp2f(log2_decay(log_decay[h]));
    const T* qp = q.p + b * q.sb + h * q.sh;
    const T* kp = k.p + b * k.sb + h * k.sh;
    const T* vp = v.p + b * v.sb + h * v.sh;
    float vv[VE], acc[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) {
        vv[e] = c + e < dim ? (float)vp[c + e] : 0.0f;
        acc[e] = 0.0f;
    }
    float* sp = state + head * dim * dim + c;
    if (c < dim) {
#pragma unroll 4
        for (int row = group; row < dim; row += kGroups) {
            const float kk = (float)kp[row], qq = (float)qp[row];
            float x[VE];
            if (VE == 1) {
                x[0] = sp[row * dim];
            } else {
                const vec r = *reinterpret_cast<const vec*>(sp + row * dim);
#pragma unroll
                for (int e = 0; e < VE; ++e) x[e] = r[e];
            }
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                x[e] = fmaf(x[e], a, kk * vv[e]);
                acc[e] = fmaf(qq, x[e], acc[e]);
            }
            if (VE == 1) {
                sp[row * dim] = x[0];
            } else {
                vec r;
#pragma unroll
                for (int e = 0; e < VE; ++e) r[e] = x[e];
                *reinterpret_cast<vec*>(sp + row * dim) = r;
            }
        }
    }
#pragma unroll
    for (int e = 0; e < VE; ++e) {
        for (int d = kLanes; d < 64; d <<= 1) acc[e] += __shfl_xor(acc[e], d);
        if ((int)(threadIdx.x & 63) < kLanes) sums[threadIdx.x >> 6][threadIdx.x % kLanes * VE + e] = acc[e];
    }
    __syncthreads();
    const int t = threadIdx.x, oc = blockIdx.x % slices * 32 + t;
    if (t < 32 && oc < dim) o[head * dim + oc] = (T)(scale * ((sums[0][t] + sums[1][t]) + (sums[2][t] + sums[3][t])));
}

constexpr int kJoinFrom = 8;

// Spans per sequence: none where the walks fill half of the chip, else as many as fill it -- a compute unit holds three
// walks of up to 64 columns, two of more -- down to one piece each.  24 ragged sequences of up to 2000 rows, 8 heads, trained
// (192 and 576 walks): 198 us, with the backward walks cut in two as well 231.  4 x 16 heads of 8192 rows: 104 us with 768
// walks, 117 with 512, 115 with 1536.  One sequence of 300 rows and 8 heads: 16 us, with spans of four pieces and more 21.
int span_count(int64_t n_seq, int64_t max_len, int64_t heads, int dim, int walks) {
    const int64_t blocks = n_seq * heads * walks, fill = dim > 64 ? 512 : 768;
    int64_t n = blocks >= 512 ? 1 : (fill + blocks - 1) / blocks;
    const int64_t most = (max_len + kPiece - 1) / kPiece;
    if (n > most) n = most;
    return (int)(n < 1 ? 1 : n);
}

template <typename T, int DP>
int allow_walks() {
    const void* f[] = {reinterpret_cast<const void*>(&decay_walk_kernel<T, DP, false, false>), reinterpret_cast<const void*>(&decay_walk_kernel<T, DP, false, true>),
                       reinterpret_cast<const void*>(&decay_walk_kernel<T, DP, true, false>), reinterpret_cast<const void*>(&decay_walk_kernel<T, DP, true, true>)};
    for (const void* k : f) VAD_HIP_CHECK(hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)WalkShape<T, DP>::kLds));
    return VAD_OK;
}

template <typename T, int DP, bool STATE>
void launch_walk(const WalkArgs<T>& a, int walks, hipStream_t st) {
    const dim3 grid((unsigned)(a.n_seq * a.heads * a.n_spans), (unsigned)walks), block((WalkShape<T, DP>::kThreads));
    constexpr size_t lds = WalkShape<T, DP>::kLds;
    if (a.whole)
        hipLaunchKernelGGL((decay_walk_kernel<T, DP, STATE, true>), grid, block, lds, st, a);
    else
        hipLaunchKernelGGL((decay_walk_kernel<T, DP, STATE, false>), grid, block, lds, st, a);
}
template <typename T, bool STATE>
void launch_walk(const WalkArgs<T>& a, int walks, hipStream_t st) {
    if (a.dim <= 32)
        launch_walk<T, 32, STATE>(a, walks, st);
    else if (a.dim <= 64)
        launch_walk<T, 64, STATE>(a, walks, st);
    else
        launch_walk<T, 128, STATE>(a, walks, st);
}

template <typename T>
int run_walks(const WalkArgs<T>& a, int walks, hipStream_t st) {
    if (a.n_spans > 1) {
        launch_walk<T, true>(a, walks, st);
        VAD_HIP_CHECK(hipGetLastError());
        if (a.joined) {
            const int64_t blocks = ((int64_t)a.dim * a.dim + 255) / 256 * a.n_seq * a.heads;
            hipLaunchKernelGGL((decay_join_kernel<T>), dim3((unsigned)blocks, (unsigned)walks), dim3(256), 0, st, a);
            VAD_HIP_CHECK(hipGetLastError());
        }
    }
    launch_walk<T, false>(a, walks, st);
    VAD_HIP_CHECK(hipGetLastError());
    return VAD_OK;
}

template <typename T>
Heads<const T> heads_of(const void* p, const int64_t* strides) {
    return {static_cast<const T*>(p), strides[0], strides[1], strides[2]};
}
template <typename T>
int run_forward(const void* q, const int64_t* qs, const void* k, const int64_t* ks, const void* v, const int64_t* vs, Sequences seq,
                int n_seq, int heads, int dim, const float* log_decay, float scale, const float* s0, void* o, float* s1, int n_spans,
                float* ws, hipStream_t st) {
    WalkArgs<T> a = {};
    a.walk[0] = {heads_of<T>(q, qs), heads_of<T>(k, ks), heads_of<T>(v, vs), static_cast<T*>(o), s0, s1, scale, scale, 1.0f, false, false};
    a.seq = seq;
    a.log_decay = log_decay;
    a.spans = n_spans > 1 ? ws : nullptr;
    a.n_seq = n_seq;
    a.heads = heads;
    a.dim = dim;
    a.n_spans = n_spans;
    a.joined = n_spans > kJoinFrom;
    a.whole = whole_rows(a.walk[0].q, dim) && whole_rows(a.walk[0].k, dim) && whole_rows(a.walk[0].v, dim) && whole_words(a.walk[0].o, dim);
    return run_walks(a, 1, st);
}

template <typename T>
int run_backward(const void* q, const int64_t* qs, const void* k, const int64_t* ks, const void* v, const int64_t* vs, const void* g,
                 const int64_t* gs, Sequences seq, int n_seq, int heads, int dim, const float* log_decay, float scale, const float* s0,
                 const float* ds1, void* dq, void* dk, void* dv, float* ds0, int n_spans, float* ws, hipStream_t st) {
    const Heads<const T> Q = heads_of<T>(q, qs), K = heads_of<T>(k, ks), V = heads_of<T>(v, vs), G = heads_of<T>(g, gs);
    WalkArgs<T> a = {};
    a.walk[0] = {G, V, K, static_cast<T*>(dq), s0, nullptr, scale, scale, 1.0f, true, false};
    a.walk[1] = {V, G, Q, static_cast<T*>(dk), ds1, nullptr, scale, 1.0f, scale, true, true};
    a.walk[2] = {K, Q, G, static_cast<T*>(dv), ds1, ds0, scale, 1.0f, scale, false, true};
    a.seq = seq;
    a.log_decay = log_decay;
    a.spans = n_spans > 1 ? ws : nullptr;
    a.n_seq = n_seq;
    a.heads = heads;
    a.dim = dim;
    a.n_spans = n_spans;
    a.joined = n_spans > kJoinFrom;
    a.whole = whole_rows(Q, dim) && whole_rows(K, dim) && whole_rows(V, dim) && whole_rows(G, dim);
    for (const Walk<T>& w : a.walk) a.whole = a.whole && whole_words(w.o, dim);
    return run_walks(a, 3, st);
}

int check_heads(int64_t n_seq, int64_t n_tokens, int64_t max_len, int heads, int dim, int dtype, float scale) {
    VAD_REQUIRE(dtype == VAD_DTYPE_F32 || dtype == VAD_DTYPE_BF16, "dtype must be VAD_DTYPE_F32 or VAD_DTYPE_BF16, got %d", dtype);
    VAD_REQUIRE(dim >= 1 && dim <= VAD_MAX_HEAD_DIM, "head dimension %d out of range 1..%d", dim, VAD_MAX_HEAD_DIM);
    VAD_REQUIRE(heads >= 1, "heads must be positive, got %d", heads);
    VAD_REQUIRE(fabsf(scale) < INFINITY, "scale must be finite in float32");
    VAD_REQUIRE(n_seq >= 0 && n_tokens >= 0 && max_len >= 0, "negative sequence count or length");
    VAD_REQUIRE(n_tokens <= (1 << 30) && max_len <= (1 << 30), "length out of range");
    // a step launches up to four blocks of 256 threads for each, and a launch's threads are counted in 32 bits
    VAD_REQUIRE(n_seq < (1 << 22) / heads, "too many sequences for one launch");
    VAD_REQUIRE((int64_t)heads * dim < VAD_MAX_ROW_STRIDE, "rows of %lld elements are too long", (long long)heads * dim);
    return VAD_OK;
}

int check_rows(const int64_t* strides) {
    VAD_REQUIRE(strides[1] >= 0 && strides[1] < VAD_MAX_ROW_STRIDE, "row stride %lld out of range", (long long)strides[1]);
    return VAD_OK;
}

}  // namespace

// The float32 walks of 33 and more columns use more than 64 KB of LDS: opt in once per device.
int ensure_linear_attention_attrs() {
    static std::mutex mu;
    static bool done[64] = {false};
    int dev = 0;
    VAD_HIP_CHECK(hipGetDevice(&dev));
    VAD_REQUIRE(dev >= 0 && dev < 64, "device index %d out of range", dev);
    std::lock_guard<std::mutex> lock(mu);
    if (done[dev]) return VAD_OK;
    int rc = VAD_OK;
    if ((rc = allow_walks<float, 32>()) != VAD_OK || (rc = allow_walks<float, 64>()) != VAD_OK || (rc = allow_walks<float, 128>()) != VAD_OK ||
        (rc = allow_walks<__bf16, 32>()) != VAD_OK || (rc = allow_walks<__bf16, 64>()) != VAD_OK || (rc = allow_walks<__bf16, 128>()) != VAD_OK)
        return rc;
    done[dev] = true;
    return VAD_OK;
}
}  // namespace vad

extern "C" size_t vad_linear_attention_workspace_bytes(int64_t n_seq, int64_t max_len, int heads, int dim, int backward) {
    using namespace vad;
    if (n_seq <= 0 || max_len <= 0 || heads <= 0 || dim <= 0) return 0;
    const int walks = backward ? 3 : 1, spans = span_count(n_seq, max_len, heads, dim, walks);
    return spans > 1 ? (size_t)walks * n_seq * heads * spans * dim * dim * sizeof(float) : 0;
}

extern "C" int vad_linear_attention_forward(const void* q_dev, const int64_t* q_strides, const void* k_dev, const int64_t* k_strides,
                                            const void* v_dev, const int64_t* v_strides, const int64_t* starts_dev, int64_t n_seq,
                                            int64_t n_tokens, int64_t max_len, int heads, int dim, int dtype,
                                            const float* log_decay_dev, float scale, const float* state_in_dev, void* o_dev,
                                            float* state_out_dev, void* workspace_dev, size_t workspace_bytes, void* stream) {
    using namespace vad;
    int rc = check_heads(n_seq, n_tokens, max_len, heads, dim, dtype, scale);
    if (rc != VAD_OK) return rc;
    VAD_REQUIRE(q_strides && k_strides && v_strides && log_decay_dev, "null pointer argument");
    if (n_seq == 0) return VAD_OK;
    const bool empty = starts_dev ? n_tokens == 0 : max_len == 0;
    VAD_REQUIRE(empty || (q_dev && k_dev && v_dev && o_dev), "null pointer argument");
    VAD_REQUIRE(!state_in_dev || state_in_dev != state_out_dev, "state_out must not be state_in");
    for (const int64_t* strides : {q_strides, k_strides, v_strides})
        if ((rc = check_rows(strides)) != VAD_OK) return rc;
    const size_t need = vad_linear_attention_workspace_bytes(n_seq, max_len, heads, dim, 0);
    VAD_REQUIRE(workspace_bytes >= need && (!need || workspace_dev), "workspace of %zu bytes is too small: %zu", workspace_bytes, need);
    rc = ensure_linear_attention_attrs();
    if (rc != VAD_OK) return rc;
    const int spans = span_count(n_seq, max_len, heads, dim, 1);
    const Sequences seq = {starts_dev, n_tokens, max_len};
    hipStream_t st = static_cast<hipStream_t>(stream);
    float* ws = static_cast<float*>(workspace_dev);
    return dtype == VAD_DTYPE_F32
               ? run_forward<float>(q_dev, q_strides, k_dev, k_strides, v_dev, v_strides, seq, (int)n_seq, heads, dim, log_decay_dev,
                                    scale, state_in_dev, o_dev, state_out_dev, spans, ws, st)
               : run_forward<__bf16>(q_dev, q_strides, k_dev, k_strides, v_dev, v_strides, seq, (int)n_seq, heads, dim, log_decay_dev,
                                     scale, state_in_dev, o_dev, state_out_dev, spans, ws, st);
}

extern "C" int vad_linear_attention_backward(const void* q_dev, const int64_t* q_strides, const void* k_dev, const int64_t* k_strides,
                                             const void* v_dev, const int64_t* v_strides, const void* do_dev, const int64_t* do_strides,
                                             const int64_t* starts_dev, int64_t n_seq, int64_t n_tokens, int64_t max_len, int heads,
                                             int dim, int dtype, const float* log_decay_dev, float scale, const float* state_in_dev,
                                             const float* dstate_out_dev, void* dq_dev, void* dk_dev, void* dv_dev,
                                             float* dstate_in_dev, void* workspace_dev, size_t workspace_bytes, void* stream) {
    using namespace vad;
    int rc = check_heads(n_seq, n_tokens, max_len, heads, dim, dtype, scale);
    if (rc != VAD_OK) return rc;
    VAD_REQUIRE(q_strides && k_strides && v_strides && do_strides && log_decay_dev, "null pointer argument");
    if (n_seq == 0) return VAD_OK;
    const bool empty = starts_dev ? n_tokens == 0 : max_len == 0;
    VAD_REQUIRE(empty || (q_dev && k_dev && v_dev && do_dev && dq_dev && dk_dev && dv_dev), "null pointer argument");
    VAD_REQUIRE(!dstate_out_dev || dstate_out_dev != dstate_in_dev, "dstate_in must not be dstate_out");
    for (const int64_t* strides : {q_strides, k_strides, v_strides, do_strides})
        if ((rc = check_rows(strides)) != VAD_OK) return rc;
    const size_t need = vad_linear_attention_workspace_bytes(n_seq, max_len, heads, dim, 1);
    VAD_REQUIRE(workspace_bytes >= need && (!need || workspace_dev), "workspace of %zu bytes is too small: %zu", workspace_bytes, need);
    rc = ensure_linear_attention_attrs();
    if (rc != VAD_OK) return rc;
    const int spans = span_count(n_seq, max_len, heads, dim, 3);
    const Sequences seq = {starts_dev, n_tokens, max_len};
    hipStream_t st = static_cast<hipStream_t>(stream);
    float* ws = static_cast<float*>(workspace_dev);
    return dtype == VAD_DTYPE_F32
               ? run_backward<float>(q_dev, q_strides, k_dev, k_strides, v_dev, v_strides, do_dev, do_strides, seq, (int)n_seq, heads,
                                     dim, log_decay_dev, scale, state_in_dev, dstate_out_dev, dq_dev, dk_dev, dv_dev, dstate_in_dev,
                                     spans, ws, st)
               : run_backward<__bf16>(q_dev, q_strides, k_dev, k_strides, v_dev, v_strides, do_dev, do_strides, seq, (int)n_seq, heads,
                                      dim, log_decay_dev, scale, state_in_dev, dstate_out_dev, dq_dev, dk_dev, dv_dev, dstate_in_dev,
                                      spans, ws, st);
}

extern "C" int vad_linear_attention_step(const void* q_dev, const int64_t* q_strides, const void* k_dev, const int64_t* k_strides,
                                         const void* v_dev, const int64_t* v_strides, int64_t batch, int heads, int dim, int dtype,
                                         const float* log_decay_dev, float scale, float* state_dev, void* o_dev, void* stream) {
    using namespace vad;
    int rc = check_heads(batch, 0, 0, heads, dim, dtype, scale);
    if (rc != VAD_OK) return rc;
    if (batch == 0) return VAD_OK;
    VAD_REQUIRE(q_dev && k_dev && v_dev && q_strides && k_strides && v_strides && log_decay_dev && state_dev && o_dev, "null pointer argument");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int slices = (dim + 31) / 32;
    const dim3 grid((unsigned)(batch * heads * slices));
    const uintptr_t at = reinterpret_cast<uintptr_t>(state_dev);
    const int ve = dim % 4 == 0 && at % 16 == 0 ? 4 : (dim % 2 == 0 && at % 8 == 0 ? 2 : 1);
    // strides here are (batch, head): Heads' row stride is not used
    const auto run = [&](auto zero) {
        typedef decltype(zero) T;
        const Heads<const T> q = {static_cast<const T*>(q_dev), q_strides[0], 0, q_strides[1]};
        const Heads<const T> k = {static_cast<const T*>(k_dev), k_strides[0], 0, k_strides[1]};
        const Heads<const T> v = {static_cast<const T*>(v_dev), v_strides[0], 0, v_strides[1]};
        T* o = static_cast<T*>(o_dev);
        if (ve == 4)
            hipLaunchKernelGGL((decay_step_kernel<T, 4>), grid, dim3(256), 0, st, q, k, v, log_decay_dev, scale, heads, dim, slices, state_dev, o);
        else if (ve == 2)
            hipLaunchKernelGGL((decay_step_kernel<T, 2>), grid, dim3(256), 0, st, q, k, v, log_decay_dev, scale, heads, dim, slices, state_dev, o);
        else
            hipLaunchKernelGGL((decay_step_kernel<T, 1>), grid, dim3(256), 0, st, q, k, v, log_decay_dev, scale, heads, dim, slices, state_dev, o);
    };
    if (dtype == VAD_DTYPE_F32)
        run(0.0f);
    else
        run((__bf16)0.0f);
    VAD_HIP_CHECK(hipGetLastError());
    return VAD_OK;
}
