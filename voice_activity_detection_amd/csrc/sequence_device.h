// Shared device code of the sequence operators (layer norm, linear attention, window attention): element types,
// 16x16 matrix tiles, and the staging of rows into LDS.
//
// One fragment type serves both element types.  A fragment is a lane's eight values of a 16 x 32 operand: lane 16 g + c
// holds row (or column) c and eight of the 32 contraction indices.  bfloat16 takes it in one v_mfma_f32_16x16x32_bf16;
// float32 in eight v_mfma_f32_16x16x4_f32, the j-th of which contracts the j-th value of every lane.  A product only
// needs both operands to use the same order of the contraction indices, and there are two:
//   natural   lane group g holds indices 8 g + j
//   split     lane group g holds 4 g + j (j < 4) and 16 + 4 g + j - 4 (j >= 4): the order in which two 16x16 result
//             tiles stacked along the contraction leave their values in the lanes, so that a result becomes the next
//             product's operand without leaving its registers.
// A result tile (float4 per lane) holds column c and rows 4 g + i.
#pragma once
#include <math.h>

#include <algorithm>

#include "vad_internal.h"

namespace vad {
namespace sq {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
// global memory takes 16-byte accesses at any 4-byte boundary
typedef u32x4 u32x4_any __attribute__((aligned(4)));
typedef u32x2 u32x2_any __attribute__((aligned(4)));

constexpr float kLog2e = 1.4426950408889634f;

template <typename T>
struct Elem;
template <>
struct Elem<float> {
    typedef f32x8 Frag;
    typedef f32x4 Quad;
    static constexpr int kPer16B = 4;
};
template <>
struct Elem<__bf16> {
    typedef bf16x8 Frag;
    typedef bf16x4 Quad;
    static constexpr int kPer16B = 8;
};
template <typename T>
using Frag = typename Elem<T>::Frag;
template <typename T>
using Quad = typename Elem<T>::Quad;

__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(f32x8 a, f32x8 b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

__device__ __forceinline__ int lane_id() { return (int)(threadIdx.x & 63); }

// ---- across lanes, without the LDS unit ----

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, false));
}
// The values that lanes i and i ^ 16 (i ^ 32) hold, the same pair in both: the swap exchanges the odd half of its first
// operand's lanes with the even half of its second's.  (The results are copied out before the cast: a bit cast of a
// vector's element reads element 0.)
template <int DISTANCE>
__device__ __forceinline__ void lane_pair(float x, float& a, float& b) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    unsigned first, second;
    if (DISTANCE == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        first = r[0], second = r[1];
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        first = r[0], second = r[1];
    }
    a = __builtin_bit_cast(float, first);
    b = __builtin_bit_cast(float, second);
}
// Sum over aligned groups of `lanes` lanes (a power of two, uniform), the same value in each.
__device__ __forceinline__ float lanes_sum(float x, int lanes) {
    if (lanes > 1) x += dpp<0xB1>(x);           // lane ^ 1
    if (lanes > 2) x += dpp<0x4E>(x);           // lane ^ 2
    if (lanes > 4) x += dpp<0x141>(x);          // the other quad of the half row
    if (lanes > 8) x += dpp<0x140>(x);          // the other half of the row
    if (lanes > 16) {
        float a, b;
        lane_pair<16>(x, a, b);
        x = a + b;
    }
    if (lanes > 32) {
        float a, b;
        lane_pair<32>(x, a, b);
        x = a + b;
    }
    return x;
}
// Over the four lanes that hold the same column of a result tile.
__device__ __forceinline__ float groups_sum(float x) {
    float a, b;
    lane_pair<16>(x, a, b);
    lane_pair<32>(a + b, a, b);
    return a + b;
}
__device__ __forceinline__ float groups_max(float x) {
    float a, b;
    lane_pair<16>(x, a, b);
    lane_pair<32>(fmaxf(a, b), a, b);
    return fmaxf(a, b);
}

// ---- rows in global memory ----

// A tensor of heads over packed or padded sequences; strides in elements, the last dimension is dense.
template <typename T>
struct Heads {
    T* p;
    int64_t sb, st, sh;
};

// The rows of sequence s: row t at p + t * st, t < len.  starts == nullptr: len = max_len rows at s * sb.  Otherwise rows
// starts[s] .. starts[s + 1] - 1 of a packed tensor of n_tokens rows; the table is not trusted: both ends are clamped.
struct Sequences {
    const int64_t* starts;
    int64_t n_tokens, max_len;
};
__device__ __forceinline__ void sequence_rows(const Sequences& q, int s, int64_t& first, int64_t& len) {
    if (!q.starts) {
        first = 0;
        len = q.max_len;
        return;
    }
    int64_t lo = q.starts[s], hi = q.starts[s + 1];
    lo = lo < 0 ? 0 : (lo > q.n_tokens ? q.n_tokens : lo);
    hi = hi < lo ? lo : (hi > q.n_tokens ? q.n_tokens : hi);
    first = lo;
    len = hi - lo;
}
// Rows of a packed output of `width` elements a row that lie before the first sequence or behind the last one become
// zero: columns c0 .. c0 + cols - 1, by the blocks of the first and the last sequence; `part` of `parts` blocks of each.
template <typename T>
__device__ __forceinline__ void zero_outside(T* out, int64_t width, int c0, int cols, const Sequences& q, int s, int n_seq, int part, int parts) {
    if (!q.starts || (s != 0 && s != n_seq - 1)) return;
    int64_t lo = q.starts[0], hi = q.starts[n_seq];
    lo = lo < 0 ? 0 : (lo > q.n_tokens ? q.n_tokens : lo);
    hi = hi < lo ? lo : (hi > q.n_tokens ? q.n_tokens : hi);
    if (s == 0)
        for (int64_t i = (int64_t)part * blockDim.x + threadIdx.x; i < lo * cols; i += (int64_t)parts * blockDim.x)
            out[i / cols * width + c0 + i % cols] = (T)0.0f;
    if (s == n_seq - 1)
        for (int64_t i = (int64_t)part * blockDim.x + threadIdx.x; i < (q.n_tokens - hi) * cols; i += (int64_t)parts * blockDim.x)
            out[(hi + i / cols) * width + c0 + i % cols] = (T)0.0f;
}

template <typename T>
__device__ __forceinline__ T* head_ptr(const Heads<T>& x, const Sequences& q, int s, int64_t first, int h) {
    return x.p + (q.starts ? first * x.st : (int64_t)s * x.sb) + (int64_t)h * x.sh;
}

// 16 bytes of a row from column c; columns from `cols` on read as zero.  `whole`: rows start at 4-byte boundaries, so that
// pieces inside the row are one load (uniform over the launch).
template <typename T>
__device__ __forceinline__ u32x4 load_piece(const T* row, int c, int cols, bool whole) {
    constexpr int VE = Elem<T>::kPer16B;
    u32x4 r;
    if (whole && c + VE <= cols) {
        r = *reinterpret_cast<const u32x4_any*>(row + c);
    } else {
        T v[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) v[e] = c + e < cols ? row[c + e] : (T)0.0f;
        __builtin_memcpy(&r, v, 16);
    }
    return r;
}

template <typename T>
__device__ __forceinline__ void store_piece(T* row, int c, int cols, u32x4 v, bool whole) {
    constexpr int VE = Elem<T>::kPer16B;
    if (whole && c + VE <= cols) {
        *reinterpret_cast<u32x4_any*>(row + c) = v;
    } else {
        T e[VE];
        __builtin_memcpy(e, &v, 16);
#pragma unroll
        for (int i = 0; i < VE; ++i)
            if (c + i < cols) row[c + i] = e[i];
    }
}

// Rows at 4-byte boundaries and of whole 4-byte words: the form that buffer loads and wide stores take.
template <typename T>
bool whole_words(const Heads<T>& x, int dim) {
    const uint64_t at = reinterpret_cast<uintptr_t>(x.p) | (uint64_t)(x.sb * sizeof(T)) | (uint64_t)(x.st * sizeof(T)) | (uint64_t)(x.sh * sizeof(T));
    return at % 4 == 0 && dim * sizeof(T) % 4 == 0;
}
// The same of rows that a buffer can end behind: it leaves out what lies behind the last row, which rows that overlap -- one
// for all, or windows over one run of values -- would find in the rows before it.
template <typename T>
bool whole_rows(const Heads<T>& x, int dim) {
    return x.st >= dim && whole_words(x, dim);
}
template <typename T>
bool whole_words(const T* p, int dim) {
    return reinterpret_cast<uintptr_t>(p) % 4 == 0 && dim * sizeof(T) % 4 == 0;
}

// A buffer over `rows` rows of `cols` columns, the last one cut at its end: loads past it give zero, without a branch.
// At most 64 rows, 2^22 elements apart (VAD_MAX_ROW_STRIDE): offsets stay below 2^30 bytes.
template <typename T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_buffer(const T* p, int64_t st, int rows, int cols) {
    const int bytes = rows > 0 ? ((rows - 1) * (int)st + cols) * (int)sizeof(T) : 0;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(p), 0, bytes, 0x00020000);
}
__device__ __forceinline__ u32x4 load_piece(__amdgpu_buffer_rsrc_t b, int offset) {
    return __builtin_amdgcn_raw_buffer_load_b128(b, offset, 0, 0);
}

// Whether any of the values in some 16-byte pieces is an infinity or a NaN.  Times zero they are NaN, and two bfloat16 take one
// instruction for that; of float32 the largest bit pattern without its sign says it.
template <typename T, int N>
__device__ __forceinline__ bool any_not_finite(const u32x4 (&v)[N]) {
    if constexpr (sizeof(T) == 4) {
        unsigned top = 0;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = max(top, v[n][i] & 0x7FFFFFFFu);
        return top >= 0x7F800000u;
    } else {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        const bf16x2 zero = {(__bf16)0.0f, (__bf16)0.0f};
        float sum = 0.0f;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned word = v[n][i];
                sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, word), zero, sum, false);
            }
        return sum != sum;
    }
}

// 64 rows of one head on their way through a block's registers into an LDS tile of PITCH elements a row.  BUF: by buffer
// loads (whole_words).
template <typename T, int DP, int NT, bool BUF, int PITCH>
struct Staged {
    static constexpr int kPer = Elem<T>::kPer16B, kPPR = DP / kPer, kLd = PITCH, kPieces = 64 * kPPR / NT, kStep = NT / kPPR;
    u32x4 r[kPieces];

    // Tile row i is row at + i of the head (`back`: at - i) for i < rows, zero from there on; uniform arguments.
    __device__ __forceinline__ void fetch(const T* p, int64_t st, int64_t at, int rows, int dim, bool back = false) {
        rows = rows < 64 ? rows : 64;
        const int row0 = threadIdx.x / kPPR, c = threadIdx.x % kPPR * kPer;
        if constexpr (BUF) {
            const auto b = row_buffer(p + (back ? at - (rows - 1) : at) * st, st, rows, dim);
            const int col = c < dim ? c * (int)sizeof(T) : 1 << 30, pitch = (int)st * (int)sizeof(T);
#pragma unroll
            for (int n = 0; n < kPieces; ++n) {
                const int row = row0 + n * kStep;
                r[n] = load_piece(b, (back ? rows - 1 - row : row) * pitch + col);
            }
        } else {
#pragma unroll
            for (int n = 0; n < kPieces; ++n) {
                const int row = row0 + n * kStep;
                r[n] = u32x4{0, 0, 0, 0};
                if (row < rows) r[n] = load_piece(p + (back ? at - row : at + row) * st, c, dim, false);
            }
        }
    }
    __device__ __forceinline__ void put(T* tile, int dim) {
        const int row0 = threadIdx.x / kPPR, c = threadIdx.x % kPPR * kPer;
        if (BUF && dim < DP) {          // a piece that crosses the row's end has read on into what follows
            const int words = (dim - c) * (int)sizeof(T) / 4;
#pragma unroll
            for (int n = 0; n < kPieces; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) r[n][i] = i < words ? r[n][i] : 0u;
        }
#pragma unroll
        for (int n = 0; n < kPieces; ++n) *reinterpret_cast<u32x4*>(tile + (row0 + n * kStep) * kLd + c) = r[n];
    }
    __device__ __forceinline__ bool not_finite() const { return any_not_finite<T>(r); }
};

// The infinities and NaN in a tile's first `rows` rows become zero: every thread of the block cleans pieces of it.
template <typename T, int DP, int NT, int PITCH>
__device__ __forceinline__ void clean_tile(T* tile, int rows) {
    using S = Staged<T, DP, NT, true, PITCH>;
    const int row0 = threadIdx.x / S::kPPR, c = threadIdx.x % S::kPPR * S::kPer;
#pragma unroll 1
    for (int n = 0; n < S::kPieces; ++n) {
        T* p = tile + (row0 + n * S::kStep) * S::kLd + c;
        if (row0 + n * S::kStep >= rows) break;
#pragma unroll
        for (int e = 0; e < S::kPer; ++e)
            if (!(fabsf((float)p[e]) < INFINITY)) p[e] = (T)0.0f;
    }
}

// ---- fragments from LDS ----

// Lane c: row r0 + c, columns c0 + 8 g + j.
template <typename T>
__device__ __forceinline__ Frag<T> frag_natural(const T* tile, int ld, int r0, int c0) {
    const int l = lane_id();
    const T* p = tile + (r0 + (l & 15)) * ld + c0 + 8 * (l >> 4);
    Frag<T> f;
    if (sizeof(T) == 2) {
        f = *reinterpret_cast<const Frag<T>*>(p);
    } else {
        const f32x4 a = reinterpret_cast<const f32x4*>(p)[0], b = reinterpret_cast<const f32x4*>(p)[1];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f[j] = a[j];
            f[j + 4] = b[j];
        }
    }
    return f;
}

// Lane c: row r0 + c, columns c0 + (4 g + j | 16 + 4 g + j - 4).
template <typename T>
__device__ __forceinline__ Frag<T> frag_split(const T* tile, int ld, int r0, int c0) {
    const int l = lane_id();
    const T* p = tile + (r0 + (l & 15)) * ld + c0 + 4 * (l >> 4);
    const Quad<T> a = *reinterpret_cast<const Quad<T>*>(p), b = *reinterpret_cast<const Quad<T>*>(p + 16);
    Frag<T> f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f[j] = a[j];
        f[j + 4] = b[j];
    }
    return f;
}

// Transposed: lane c: column c0 + c, rows r0 + (4 g + j | 16 + 4 g + j - 4).  The 16-bit form uses the LDS read that
// transposes a 4 x 16 block within each group of 16 lanes (lane i supplies the address of row i >> 2, columns
// 4 (i & 3) .. + 3 and receives column i of the four rows).
__device__ __forceinline__ bf16x8 frag_columns(const __bf16* tile, int ld, int r0, int c0) {
    typedef __attribute__((address_space(3))) s16x4* lds_ptr;
    const int l = lane_id();
    const __bf16* p = tile + (r0 + 4 * (l >> 4) + ((l >> 2) & 3)) * ld + c0 + 4 * (l & 3);
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)p);
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 16 * ld));
    bf16x8 f;
    __builtin_memcpy(&f, &a, 8);
    __builtin_memcpy(reinterpret_cast<char*>(&f) + 8, &b, 8);
    return f;
}
__device__ __forceinline__ f32x8 frag_columns(const float* tile, int ld, int r0, int c0) {
    const int l = lane_id();
    const float* p = tile + (r0 + 4 * (l >> 4)) * ld + c0 + (l & 15);
    f32x8 f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f[j] = p[j * ld];
        f[j + 4] = p[(16 + j) * ld];
    }
    return f;
}

// Two stacked result tiles as an operand in split order.
__device__ __forceinline__ void to_frag(f32x4 a, f32x4 b, bf16x8& f) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f[j] = (__bf16)a[j];
        f[j + 4] = (__bf16)b[j];
    }
}
__device__ __forceinline__ void to_frag(f32x4 a, f32x4 b, f32x8& f) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f[j] = a[j];
        f[j + 4] = b[j];
    }
}

// Four consecutive values of an output row; `whole`: rows start at 4-byte boundaries.
template <typename T>
__device__ __forceinline__ void store_quad(T* row, int c, int cols, f32x4 v, bool whole) {
    T q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = (T)v[i];
    if (whole && c + 4 <= cols) {
        if (sizeof(T) == 4) {
            u32x4 r;
            __builtin_memcpy(&r, q, 16);
            *reinterpret_cast<u32x4_any*>(row + c) = r;
        } else {
            u32x2 r;
            __builtin_memcpy(&r, q, 8);
            *reinterpret_cast<u32x2_any*>(row + c) = r;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c + i < cols) row[c + i] = q[i];
    }
}

}  // namespace sq
}  // namespace vad
