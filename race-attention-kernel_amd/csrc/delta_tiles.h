// delta_tiles.h -- device helpers of the gated delta rule's chunk kernels
// (delta_chunk.hip, delta_bwd.hip): 64-token tiles in LDS and the order of
// matrix-core operands.  Not part of the ABI.
//
// Operands.  bf16 rows run on v_mfma_f32_16x16x32_bf16; what is computed from
// them enters a product rounded to bf16 (One) or as a bf16 hi + lo pair (Two:
// 16 bits, lo * lo left out).  fp32 rows run on v_mfma_f32_16x16x4_f32 as they
// are, eight steps for the same 32 values.
//
// Order.  A lane of a wave has group g = lane / 16 and index lr = lane % 16.  A
// fragment holds 8 consecutive values of the contraction index, 32 kk + 8 g + e,
// of one row (or column) lr.  Two accumulator blocks that stand for 32 rows are
// numbered so that a lane's 4 + 4 values are such a run as well: row m = 4 q + j
// of block h (0, 1) of the pair kk is
//     tok(2 kk + h, m) = 32 kk + 8 q + 4 (h ^ (q & 1)) + j,
// so a product's accumulators are the next product's operand without leaving the
// registers (odd groups swap the halves).  h ^ (q & 1) instead of h spreads a
// transposed read over all banks.
//
// Tiles hold rows of K = 64 or 128 values, 16-byte chunk u of row r at chunk
// u ^ swizzle(r): fragment reads (16 rows tok(b, 0..15), one chunk) and
// transposed reads touch every bank once.
#pragma once

#include <initializer_list>

#include "mfma_common.h"

namespace race {
namespace delta {

using mfma::bf16x8;
using mfma::f32x4;

constexpr int kChunk = 64;  // tokens of a chunk

__device__ __forceinline__ constexpr int tok(int b, int m) {
    return 32 * (b >> 1) + 8 * (m >> 2) + 4 * ((b & 1) ^ ((m >> 2) & 1)) + (m & 3);
}

// ---- operands ----

template <typename TIn>
struct OneT;
template <typename TIn>
struct TwoT;
template <>
struct OneT<bf16_t> {
    bf16x8 h;
};
template <>
struct TwoT<bf16_t> {
    bf16x8 h, l;
};
template <>
struct OneT<float> {
    f32x4 a, b;
};
template <>
struct TwoT<float> : OneT<float> {};

__device__ __forceinline__ f32x4 mac(const OneT<bf16_t>& x, const OneT<bf16_t>& y, f32x4 acc) {
    return mfma::mfma16(x.h, y.h, acc);
}
__device__ __forceinline__ f32x4 mac(const OneT<bf16_t>& x, const TwoT<bf16_t>& y, f32x4 acc) {
    return mfma::mfma16(x.h, y.h, mfma::mfma16(x.h, y.l, acc));
}
__device__ __forceinline__ f32x4 mac(const TwoT<bf16_t>& x, const TwoT<bf16_t>& y, f32x4 acc) {
    return mfma::mfma16(x.h, y.h, mfma::mfma16(x.h, y.l, mfma::mfma16(x.l, y.h, acc)));
}
__device__ __forceinline__ f32x4 mac(const OneT<float>& x, const OneT<float>& y, f32x4 acc) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = mfma::mfma4(x.a[e], y.a[e], acc);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = mfma::mfma4(x.b[e], y.b[e], acc);
    return acc;
}

__device__ __forceinline__ OneT<bf16_t> first(const TwoT<bf16_t>& x) { return {x.h}; }
__device__ __forceinline__ OneT<float> first(const TwoT<float>& x) { return x; }

// A block pair's accumulators as operands.
__device__ __forceinline__ bf16x8 swapped(uint2 x0, uint2 x1, bool odd) {
    return __builtin_bit_cast(bf16x8, make_uint4(odd ? x1.x : x0.x, odd ? x1.y : x0.y, odd ? x0.x : x1.x, odd ? x0.y : x1.y));
}
__device__ __forceinline__ void operand(const f32x4& x0, const f32x4& x1, bool odd, OneT<bf16_t>& out) {
    uint2 h0, h1, none;
    mfma::split4<false>(x0[0], x0[1], x0[2], x0[3], h0, none);
    mfma::split4<false>(x1[0], x1[1], x1[2], x1[3], h1, none);
    out.h = swapped(h0, h1, odd);
}
__device__ __forceinline__ void operand(const f32x4& x0, const f32x4& x1, bool odd, TwoT<bf16_t>& out) {
    uint2 h0, h1, l0, l1;
    mfma::split4<true>(x0[0], x0[1], x0[2], x0[3], h0, l0);
    mfma::split4<true>(x1[0], x1[1], x1[2], x1[3], h1, l1);
    out.h = swapped(h0, h1, odd);
    out.l = swapped(l0, l1, odd);
}
__device__ __forceinline__ void operand(const f32x4& x0, const f32x4& x1, bool odd, OneT<float>& out) {
#pragma unroll
    for (int e = 0; e < 4; ++e) out.a[e] = odd ? x1[e] : x0[e], out.b[e] = odd ? x0[e] : x1[e];
}

// A fragment to memory: 8 consecutive values.
__device__ __forceinline__ void store_run(bf16_t* p, const OneT<bf16_t>& x) { *reinterpret_cast<bf16x8*>(p) = x.h; }
__device__ __forceinline__ void store_run(float* p, const OneT<float>& x) {
    *reinterpret_cast<f32x4*>(p) = x.a;
    *reinterpret_cast<f32x4*>(p + 4) = x.b;
}

// ---- tiles ----

template <typename E, int K>
struct Tile {
    static constexpr int kRow = K * int(sizeof(E));  // bytes
    static constexpr int kChunks = kRow / 16;
    static constexpr int kBytes = kChunk * kRow;
    __device__ __forceinline__ static int at(int r, int u) {
        static_assert(kRow == 128 || kRow == 256 || kRow == 512, "");
        if constexpr (sizeof(E) == 4 && kRow > 128)
            return r * kRow + 16 * (u ^ (((r >> 4) & 1) | ((r << 1) & 6) | (r & 8)));
        else if constexpr (kRow == 256)
            return r * kRow + 16 * (u ^ ((r & 1) | ((r >> 3) & 2) | ((r >> 1) & 4) | ((r << 2) & 8)));
        else
            return r * kRow + 16 * (u ^ (((r >> 1) & 1) | ((r >> 3) & 2) | ((r >> 1) & 4)));
    }
    // Values 8 u .. 8 u + 7 of a row.
    __device__ __forceinline__ static OneT<E> one(const unsigned char* t, int row, int u) {
        if constexpr (sizeof(E) == 4)
            return {*reinterpret_cast<const f32x4*>(t + at(row, 2 * u)), *reinterpret_cast<const f32x4*>(t + at(row, 2 * u + 1))};
        else
            return {*reinterpret_cast<const bf16x8*>(t + at(row, u))};
    }
    // The same of a tile in two planes (bf16), or of fp32 values.
    __device__ __forceinline__ static TwoT<E> two(const unsigned char* t, int row, int u) {
        TwoT<E> x;
        if constexpr (sizeof(E) == 4) {
            const OneT<E> o = one(t, row, u);
            x.a = o.a, x.b = o.b;
        } else {
            x.h = one(t, row, u).h, x.l = one(t + kBytes, row, u).h;
        }
        return x;
    }
    // Four rows from `row` of one column: of the 16 lanes of a group, lane 4 r + q
    // names the four columns from `col` in row r, and lane i gets column i of the 16.
    __device__ __forceinline__ static uint2 read_tr(const unsigned char* t, int row, int col) {
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        const unsigned char* p = t + at(row, col >> 3) + 8 * ((col >> 2) & 1);
        return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p)));
    }
    __device__ __forceinline__ static float value(const unsigned char* t, int row, int col) {
        return *reinterpret_cast<const float*>(t + at(row, col >> 2) + 4 * (col & 3));
    }
    // Values of rows row0 + 8 g + e, e = 0 .. 7, in column c(lr) of 16: c(4 q + j) = cols(q) + j.
    template <typename F>
    __device__ __forceinline__ static OneT<E> column(const unsigned char* t, int row0, int g, int lr, F cols) {
        OneT<E> x;
        if constexpr (sizeof(E) == 4) {
            const int col = cols(lr >> 2) + (lr & 3);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x.a[e] = value(t, row0 + 8 * g + e, col);
                x.b[e] = value(t, row0 + 8 * g + 4 + e, col);
            }
        } else {
            const int row = row0 + 8 * g + (lr >> 2), col = cols(lr & 3);
            const uint2 a = read_tr(t, row, col), b = read_tr(t, row + 4, col);
            x.h = __builtin_bit_cast(bf16x8, make_uint4(a.x, a.y, b.x, b.y));
        }
        return x;
    }
    // Of the columns tok(b, 0..15).
    __device__ __forceinline__ static OneT<E> transposed(const unsigned char* t, int row0, int b, int g, int lr) {
        return column(t, row0, g, lr, [&](int q) { return tok(b, 4 * q); });
    }
    // The same of a tile in two planes.
    __device__ __forceinline__ static TwoT<E> transposed_two(const unsigned char* t, int row0, int b, int g, int lr) {
        TwoT<E> x;
        const OneT<E> o = transposed(t, row0, b, g, lr);
        if constexpr (sizeof(E) == 4)
            x.a = o.a, x.b = o.b;
        else
            x.h = o.h, x.l = transposed(t + kBytes, row0, b, g, lr).h;
        return x;
    }
    // Values col .. col + 3 (a multiple of 4) of a row.
    __device__ __forceinline__ static f32x4 four(const unsigned char* t, int row, int col) {
        if constexpr (sizeof(E) == 4) {
            return *reinterpret_cast<const f32x4*>(t + at(row, col >> 2));
        } else {
            const uint2 u = *reinterpret_cast<const uint2*>(t + at(row, col >> 3) + 8 * ((col >> 2) & 1));
            return f32x4{mfma::lo_half(u.x), mfma::hi_half(u.x), mfma::lo_half(u.y), mfma::hi_half(u.y)};
        }
    }
    __device__ __forceinline__ static void put4(unsigned char* t, int row, int col, const f32x4& x) {
        if constexpr (sizeof(E) == 4)
            *reinterpret_cast<f32x4*>(t + at(row, col >> 2)) = x;
        else
            *reinterpret_cast<uint2*>(t + at(row, col >> 3) + 8 * ((col >> 2) & 1)) =
                make_uint2(mfma::pack2(x[0], x[1]), mfma::pack2(x[2], x[3]));
    }
    // Rows tok(b, 4 g .. 4 g + 3) of column c0 + lr, in accumulator order.
    __device__ __forceinline__ static f32x4 block(const unsigned char* t, int b, int c0, int g, int lr) {
        const int row = tok(b, 4 * g);
        if constexpr (sizeof(E) == 4) {
            return f32x4{value(t, row, c0 + lr), value(t, row + 1, c0 + lr), value(t, row + 2, c0 + lr), value(t, row + 3, c0 + lr)};
        } else {
            const uint2 u = read_tr(t, row + (lr >> 2), c0 + 4 * (lr & 3));
            return f32x4{mfma::lo_half(u.x), mfma::hi_half(u.x), mfma::lo_half(u.y), mfma::hi_half(u.y)};
        }
    }
};
// Bytes of a tile that two() reads.
template <typename E, int K>
constexpr int kTwoBytes = sizeof(E) == 4 ? Tile<E, K>::kBytes : 2 * Tile<E, K>::kBytes;

// Eight consecutive values of a row, of which the first `n` are there.
template <typename TIn>
struct Eight {
    static constexpr int kVecs = int(sizeof(TIn)) / 2;
    uint4 v[kVecs];
    __device__ __forceinline__ void load(const TIn* p, int n, bool vec) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) v[i] = make_uint4(0, 0, 0, 0);
        if (n <= 0) return;
        if (vec) {
            v[0] = reinterpret_cast<const uint4*>(p)[0];
            if constexpr (kVecs == 2) {
                if (n > 4) v[1] = reinterpret_cast<const uint4*>(p)[1];
            }
        } else {
            uint32_t w[4 * kVecs];
#pragma unroll
            for (int i = 0; i < 4 * kVecs; ++i) w[i] = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (i >= n) break;
                if constexpr (kVecs == 2)
                    w[i] = __float_as_uint(p[i]);
                else
                    w[i >> 1] |= uint32_t(p[i]) << (16 * (i & 1));
            }
#pragma unroll
            for (int i = 0; i < kVecs; ++i) v[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        }
    }
};

// 64 rows of K values: each thread's 8-value pieces in registers and then in a tile.
template <typename TIn, int K, int NT>
struct Stage {
    static constexpr int kPer = kChunk * (K / 8) / NT;
    Eight<TIn> x[kPer];
    // Rows of p by stride, `live` of them there, `width` values each.
    __device__ __forceinline__ void load(const TIn* p, int64_t stride, int live, int width, bool vec) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int q = int(threadIdx.x) + i * NT, row = q / (K / 8), u = q % (K / 8);
            x[i].load(p + row * stride + 8 * u, row < live ? width - 8 * u : 0, vec);
        }
    }
    __device__ __forceinline__ void put(unsigned char* t) const {
        constexpr int kVecs = Eight<TIn>::kVecs;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int q = int(threadIdx.x) + i * NT, row = q / (K / 8), u = q % (K / 8);
#pragma unroll
            for (int j = 0; j < kVecs; ++j)
                *reinterpret_cast<uint4*>(t + Tile<TIn, K>::at(row, kVecs * u + j)) = x[i].v[j];
        }
    }
};

// Dense rows of K values in memory, ROWS of them, to tiles of 64 rows one after another.
template <typename E, int K, int ROWS, int NT>
struct StageDense {
    static constexpr int kChunks = Tile<E, K>::kChunks, kPer = ROWS * kChunks / NT;
    uint4 x[kPer];
    __device__ __forceinline__ void load(const E* p) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) x[i] = reinterpret_cast<const uint4*>(p)[int(threadIdx.x) + i * NT];
    }
    __device__ __forceinline__ void put(unsigned char* t) const {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int q = int(threadIdx.x) + i * NT;
            *reinterpret_cast<uint4*>(t + Tile<E, K>::at(q / kChunks, q % kChunks)) = x[i];
        }
    }
};

// Rows of two planes (bf16), or of fp32 values, in memory and as a tile that two() reads.
template <typename E>
constexpr int kTwoRows = sizeof(E) == 4 ? kChunk : 2 * kChunk;

// ---- what the kernels share ----

constexpr double kLog2e = 1.4426950408889634074;

struct DeltaArgs {
    const void *q, *k, *v, *gate, *beta;
    const float* state;
    void* out;
    float* final_state;
    void *tm, *mm;  // [N][chunks] of T (two planes of bf16, or fp32) and M, [64][64]
    float* vec;     // [N][chunks][128]: E, then Z b
    void *st, *yt;  // nullable: [N][chunks][dvp] columns of S [DK] and Y [64], in the rows' type
    int64_t N, T;
    int64_t qn, qt, kn, kt, vn, vt;
    Live live;
    int group, dk, dv, dvp, chunks;  // group: value streams of a key stream
    int gate_f32, form;
    int vec_k, vec_v, vec_o, vec_o8;  // rows in 16-byte pieces (q and k, v; out and dout in 4 values, and whole)
    float scale;
};

// Log decays below this are taken as this: e^-200 is zero in 32 bits, and a sum
// of them still has digits for what follows.
constexpr float kLowestLog = -200.f;

__device__ __forceinline__ float gate_value(const void* p, int64_t i, int f32) {
    return f32 ? static_cast<const float*>(p)[i] : to_f32(static_cast<const bf16_t*>(p)[i]);
}
__device__ __forceinline__ float log_decay(float g, int form) {
    const float l = form == RACE_GATE_LOG ? g : fminf(g, 0.f) - log1pf(expf(-fabsf(g)));
    return l < kLowestLog ? kLowestLog : l;
}

// Four values to memory, next to each other.
__device__ __forceinline__ void store4_of(float* p, const f32x4& x) { *reinterpret_cast<f32x4*>(p) = x; }
__device__ __forceinline__ void store4_of(bf16_t* p, const f32x4& x) {
    *reinterpret_cast<uint2*>(p) = make_uint2(mfma::pack2(x[0], x[1]), mfma::pack2(x[2], x[3]));
}

// A chunk's tiles in LDS (bytes from its buffer's start).
template <typename TIn, int DK>
struct ChunkLds {
    static constexpr int kK = 0, kQ = Tile<TIn, DK>::kBytes, kT = 2 * kQ, kM = kT + kTwoBytes<TIn, 64>;
    static constexpr int kV = kM + Tile<TIn, 64>::kBytes, kVec = kV + Tile<TIn, 64>::kBytes, kBytes = kVec + 512;
    // Two buffers, where they leave the workgroup its LDS: one barrier a chunk.
    static constexpr int kBuffers = 2 * kBytes <= kGfx950LdsBytes ? 2 : 1;
};

// Consecutive streams on different XCDs, a stream's column blocks on one (they
// read the same tiles): workgroups go to the XCDs in turn.
__device__ __forceinline__ bool stream_and_block(int64_t N, int blocks, int64_t& n, int& cb) {
    const int64_t id = blockIdx.x, eight = id / (8 * blocks);
    const int in = int(id - eight * 8 * blocks);
    n = eight * 8 + (in & 7), cb = in >> 3;
    return n < N;
}

// ---- host ----

inline int dk_padded(const DeltaRule& r) { return r.dk <= 64 ? 64 : 128; }

inline bool whole_pieces(const DeltaRule& r, int64_t width, std::initializer_list<int64_t> strides) {
    const int v = r.dtype == RACE_BF16 ? 8 : 4;
    if (width % v != 0) return false;
    for (int64_t s : strides)
        if (s % v != 0) return false;
    return true;
}

inline DeltaArgs delta_args(const DeltaRule& r, const DeltaInputs& in) {
    DeltaArgs a = {};
    a.q = in.q, a.k = in.k, a.v = in.v, a.gate = in.gate, a.beta = in.beta;
    a.N = r.N, a.T = r.T;
    a.qn = r.qn, a.qt = r.qt, a.kn = r.kn, a.kt = r.kt, a.vn = r.vn, a.vt = r.vt;
    a.live = r.live;
    a.group = r.Nk > 0 ? int(r.N / r.Nk) : 1;
    a.dk = r.dk, a.dv = r.dv, a.dvp = (r.dv + 15) / 16 * 16, a.chunks = int(delta_chunks(r));
    a.gate_f32 = r.gate_dtype == RACE_F32, a.form = r.form;
    a.vec_k = whole_pieces(r, r.dk, {r.qn, r.qt, r.kn, r.kt});
    a.vec_v = whole_pieces(r, r.dv, {r.vn, r.vt});
    a.vec_o = r.dv % 4 == 0;
    a.vec_o8 = whole_pieces(r, r.dv, {});
    a.scale = r.scale;
    return a;
}

inline int64_t round256(int64_t bytes) { return (bytes + 255) / 256 * 256; }

}  // namespace delta
}  // namespace race
