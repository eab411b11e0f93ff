// delta_tiles.h -- device helpers of the gated delta rule's chunk kernels
// (delta_chunk.hip, delta_bwd.hip): 64-token tiles in LDS and the order of
// matrix-core operands.  Not part of the ABI.
//
// Operands.  bf16 rows run on v_mfma_f32_16x16x32_bf16 as they are (One); what is
// computed from them in 32 bits enters a product as three bf16 parts whose sum it is
// (Three: 24 bits; the products of parts below 2^-24 are left out), or as the first
// two (Two: 16 bits) where the result is rounded to bf16 right away.  fp32 rows run
// on v_mfma_f32_16x16x4_f32 as they are, eight steps for the same 32 values: sixteen
// times the matrix time of one bf16 product, 2.7 times that of the six of Three by Three.
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

// P bf16 parts of fp32 values, each the rounding of what the parts before leave.
template <typename TIn, int P>
struct PartsT;
template <int P>
struct PartsT<bf16_t, P> {
    bf16x8 p[P];
};
template <int P>
struct PartsT<float, P> {
    f32x4 a, b;
};
template <typename TIn>
using OneT = PartsT<TIn, 1>;
template <typename TIn>
using TwoT = PartsT<TIn, 2>;
template <typename TIn>
using ThreeT = PartsT<TIn, 3>;

// Small products first.
template <int PX, int PY>
__device__ __forceinline__ f32x4 mac(const PartsT<bf16_t, PX>& x, const PartsT<bf16_t, PY>& y, f32x4 acc) {
    constexpr int kMost = PX > PY ? PX : PY;
#pragma unroll
    for (int s = kMost - 1; s >= 0; --s)
#pragma unroll
        for (int i = 0; i < PX; ++i)
            if (s - i >= 0 && s - i < PY) acc = mfma::mfma16(x.p[i], y.p[s - i], acc);
    return acc;
}
template <int PX, int PY>
__device__ __forceinline__ f32x4 mac(const PartsT<float, PX>& x, const PartsT<float, PY>& y, f32x4 acc) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = mfma::mfma4(x.a[e], y.a[e], acc);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = mfma::mfma4(x.b[e], y.b[e], acc);
    return acc;
}

// The first Q parts.
template <int Q, int P>
__device__ __forceinline__ PartsT<bf16_t, Q> first(const PartsT<bf16_t, P>& x) {
    PartsT<bf16_t, Q> y;
#pragma unroll
    for (int i = 0; i < Q; ++i) y.p[i] = x.p[i];
    return y;
}
template <int Q, int P>
__device__ __forceinline__ PartsT<float, Q> first(const PartsT<float, P>& x) {
    return {x.a, x.b};
}

// The next part of four values, which keep what it leaves.
__device__ __forceinline__ uint2 take_part(f32x4& x) {
    const uint2 h = make_uint2(mfma::pack2(x[0], x[1]), mfma::pack2(x[2], x[3]));
    x -= f32x4{mfma::lo_half(h.x), mfma::hi_half(h.x), mfma::lo_half(h.y), mfma::hi_half(h.y)};
    return h;
}

// A block pair's accumulators as operands.
__device__ __forceinline__ bf16x8 swapped(uint2 x0, uint2 x1, bool odd) {
    return __builtin_bit_cast(bf16x8, make_uint4(odd ? x1.x : x0.x, odd ? x1.y : x0.y, odd ? x0.x : x1.x, odd ? x0.y : x1.y));
}
template <int P>
__device__ __forceinline__ void operand(const f32x4& x0, const f32x4& x1, bool odd, PartsT<bf16_t, P>& out) {
    if constexpr (P < 2) {
        f32x4 y0 = x0, y1 = x1;
        out.p[0] = swapped(take_part(y0), take_part(y1), odd);
    } else {  // fewer moves than swapping every part
        f32x4 y0, y1;
#pragma unroll
        for (int e = 0; e < 4; ++e) y0[e] = odd ? x1[e] : x0[e], y1[e] = odd ? x0[e] : x1[e];
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const uint2 h0 = take_part(y0), h1 = take_part(y1);
            out.p[i] = __builtin_bit_cast(bf16x8, make_uint4(h0.x, h0.y, h1.x, h1.y));
        }
    }
}
template <int P>
__device__ __forceinline__ void operand(const f32x4& x0, const f32x4& x1, bool odd, PartsT<float, P>& out) {
#pragma unroll
    for (int e = 0; e < 4; ++e) out.a[e] = odd ? x1[e] : x0[e], out.b[e] = odd ? x0[e] : x1[e];
}

// A fragment to memory: 8 consecutive values.
__device__ __forceinline__ void store_run(bf16_t* p, const OneT<bf16_t>& x) { *reinterpret_cast<bf16x8*>(p) = x.p[0]; }
__device__ __forceinline__ void store_run(float* p, const OneT<float>& x) {
    *reinterpret_cast<f32x4*>(p) = x.a;
    *reinterpret_cast<f32x4*>(p + 4) = x.b;
}
// A block pair's accumulators as such a run; `x` is their operand (fp32: that run).
template <int P>
__device__ __forceinline__ void store_run(float* p, const f32x4& x0, const f32x4& x1, bool odd, const PartsT<bf16_t, P>&) {
    OneT<float> run;
    operand(x0, x1, odd, run);
    store_run(p, run);
}
template <int P>
__device__ __forceinline__ void store_run(float* p, const f32x4&, const f32x4&, bool, const PartsT<float, P>& x) {
    store_run(p, first<1>(x));
}

// A wall the scheduler moves nothing across.  The walks have one wave a SIMD:
// nothing hides a read's latency but the wave's own instructions, and left alone
// the compiler puts each LDS read right in front of its product.  A stage's reads
// are issued before the products of the stage before it.
__device__ __forceinline__ void stage_wall() { __builtin_amdgcn_sched_barrier(0); }

// ---- sums over lanes, by data-parallel moves within the vector ALU ----

template <int kCtrl, int kRows>
__device__ __forceinline__ float moved(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), kCtrl, kRows, 0xf, true));
}
template <int kCtrl, int kRows>
__device__ __forceinline__ double moved(double x) {
    const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(x), kCtrl, kRows, 0xf, true);
    const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(x), kCtrl, kRows, 0xf, true);
    return __hiloint2double(hi, lo);
}
// Over the 16 lanes of a row so far: lane 15 of each has its sum.
template <typename F>
__device__ __forceinline__ F row_scan(F x) {
    x += moved<0x111, 0xf>(x);  // shifts by 1, 2, 4 and 8 lanes, zeros from outside
    x += moved<0x112, 0xf>(x);
    x += moved<0x114, 0xf>(x);
    return x + moved<0x118, 0xf>(x);
}
// Inclusive, over the 64 lanes: then the last lanes of the rows and halves before.
template <typename F>
__device__ __forceinline__ F wave_scan(F x) {
    x = row_scan(x);
    x += moved<0x142, 0xa>(x);
    return x + moved<0x143, 0xc>(x);
}
__device__ __forceinline__ float wave_sum(float x) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wave_scan(x)), 63));
}

// ---- tiles ----

// Offsets come in two parts: a lane's own (`..._base`, the same for every chunk)
// and what a product adds to it, which does not depend on the lane: rows of a
// block pair by addition, columns by exclusive or.
template <typename E, int K>
struct Tile {
    static constexpr int kRow = K * int(sizeof(E));  // bytes
    static constexpr int kChunks = kRow / 16;
    static constexpr int kBytes = kChunk * kRow;
    static constexpr int kRun = 32 * int(sizeof(E));  // bytes of 32 values
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
    __device__ __forceinline__ static int run_at(int row, int u) { return at(row, int(sizeof(E)) / 2 * u); }
    __device__ __forceinline__ static OneT<E> load(const unsigned char* t, int off) {
        if constexpr (sizeof(E) == 4)
            return {*reinterpret_cast<const f32x4*>(t + off), *reinterpret_cast<const f32x4*>(t + (off ^ 16))};
        else
            return {{*reinterpret_cast<const bf16x8*>(t + off)}};
    }
    // Row lr of block b (rows tok(b, .)), values 32 i + 8 g .., from row_base.
    __device__ __forceinline__ static int row_base(int lr, int g) { return run_at(tok(0, lr), g); }
    __device__ __forceinline__ static int row_off(int base, int b, int i) {
        return (base ^ (4 * (b & 1) * kRow) ^ (kRun * i)) + (b >> 1) * 32 * kRow;
    }
    __device__ __forceinline__ static OneT<E> one(const unsigned char* t, int base, int b, int i) {
        return load(t, row_off(base, b, i));
    }
    // The same of a tile in P planes of parts, PLANE bytes apart (bf16), or of fp32 values.
    template <int P, int PLANE = kBytes>
    __device__ __forceinline__ static PartsT<E, P> parts(const unsigned char* t, int base, int b, int i) {
        PartsT<E, P> x;
        if constexpr (sizeof(E) == 4) {
            const OneT<E> o = one(t, base, b, i);
            x.a = o.a, x.b = o.b;
        } else {
#pragma unroll
            for (int p = 0; p < P; ++p) x.p[p] = one(t + p * PLANE, base, b, i).p[0];
        }
        return x;
    }
    // Four rows of one column: of the 16 lanes of a group, lane 4 r + q names four
    // columns of row r, and lane i gets column i of the 16.
    __device__ __forceinline__ static uint2 read_tr(const unsigned char* p) {
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p)));
    }
    // Column tok(b, lr), rows 32 kk + 8 g + e, from column_base.
    __device__ __forceinline__ static int column_base(int lr, int g) {
        if constexpr (sizeof(E) == 4) {
            const int col = tok(0, lr);
            return at(8 * g, col >> 2) + 4 * (col & 3);
        } else {
            return at(8 * g + (lr >> 2), lr & 3) + 8 * (lr & 1);
        }
    }
    __device__ __forceinline__ static OneT<E> transposed(const unsigned char* t, int base, int kk, int b) {
        OneT<E> x;
        const int off = (base ^ (kRun * (b >> 1)) ^ (4 * int(sizeof(E)) * (b & 1))) + 32 * kk * kRow;
        if constexpr (sizeof(E) == 4) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x.a[e] = *reinterpret_cast<const float*>(t + (off ^ (32 * e)) + e * kRow);
                x.b[e] = *reinterpret_cast<const float*>(t + (off ^ (32 * e)) + (e + 4) * kRow);
            }
        } else {
            const uint2 a = read_tr(t + off), c = read_tr(t + off + 4 * kRow);
            x.p[0] = __builtin_bit_cast(bf16x8, make_uint4(a.x, a.y, c.x, c.y));
        }
        return x;
    }
    // The same of a tile in P planes.
    template <int P, int PLANE = kBytes>
    __device__ __forceinline__ static PartsT<E, P> transposed_parts(const unsigned char* t, int base, int kk, int b) {
        PartsT<E, P> x;
        if constexpr (sizeof(E) == 4) {
            const OneT<E> o = transposed(t, base, kk, b);
            x.a = o.a, x.b = o.b;
        } else {
#pragma unroll
            for (int p = 0; p < P; ++p) x.p[p] = transposed(t + p * PLANE, base, kk, b).p[0];
        }
        return x;
    }
    // Values col .. col + 3 (a multiple of 4) of a row.
    __device__ __forceinline__ static int four_at(int row, int col) {
        if constexpr (sizeof(E) == 4) return at(row, col >> 2);
        return at(row, col >> 3) + 8 * ((col >> 2) & 1);
    }
    __device__ __forceinline__ static f32x4 four(const unsigned char* t, int off) {
        if constexpr (sizeof(E) == 4) {
            return *reinterpret_cast<const f32x4*>(t + off);
        } else {
            const uint2 u = *reinterpret_cast<const uint2*>(t + off);
            return f32x4{mfma::lo_half(u.x), mfma::hi_half(u.x), mfma::lo_half(u.y), mfma::hi_half(u.y)};
        }
    }
    __device__ __forceinline__ static void put4(unsigned char* t, int off, const f32x4& x) {
        if constexpr (sizeof(E) == 4)
            *reinterpret_cast<f32x4*>(t + off) = x;
        else
            *reinterpret_cast<uint2*>(t + off) = make_uint2(mfma::pack2(x[0], x[1]), mfma::pack2(x[2], x[3]));
    }
    // Four fp32 values in P planes of parts (bf16), or as they are.
    template <int P, int PLANE = kBytes>
    __device__ __forceinline__ static void put4_parts(unsigned char* t, int off, f32x4 x) {
        if constexpr (sizeof(E) == 4) {
            *reinterpret_cast<f32x4*>(t + off) = x;
        } else {
#pragma unroll
            for (int p = 0; p < P; ++p) *reinterpret_cast<uint2*>(t + p * PLANE + off) = take_part(x);
        }
    }
    // Rows tok(b, 4 g .. 4 g + 3) of column c0 + lr, in accumulator order, from block_base.
    __device__ __forceinline__ static int block_base(int c0, int lr, int g) {
        const int row = tok(0, 4 * g);
        if constexpr (sizeof(E) == 4) return at(row, (c0 + lr) >> 2) + 4 * (lr & 3);
        const int col = c0 + 4 * (lr & 3);
        return at(row + (lr >> 2), col >> 3) + 8 * ((col >> 2) & 1);
    }
    __device__ __forceinline__ static f32x4 block(const unsigned char* t, int base, int b) {
        const int off = (base ^ (4 * (b & 1) * kRow)) + (b >> 1) * 32 * kRow;
        if constexpr (sizeof(E) == 4) {
            f32x4 x;
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = *reinterpret_cast<const float*>(t + (off ^ (32 * r)) + r * kRow);
            return x;
        } else {
            const uint2 u = read_tr(t + off);
            return f32x4{mfma::lo_half(u.x), mfma::hi_half(u.x), mfma::lo_half(u.y), mfma::hi_half(u.y)};
        }
    }
};
// Bytes of a tile in P planes.
template <typename E, int K, int P>
constexpr int kPartsBytes = (sizeof(E) == 4 ? 1 : P) * Tile<E, K>::kBytes;

// Eight consecutive values of a row.
template <typename TIn>
struct Eight {
    static constexpr int kVecs = int(sizeof(TIn)) / 2;
    uint4 v[kVecs];
};

// Eight values of a row, from column c on, wherever the row starts: zeros from its
// `width` on, and a row that is not there is one of zeros.  It is at element `at` of a
// view.  Offsets past the view's end stand for what is not there (a branch
// would wait for every load), and what has come is put in place when it is wanted.
template <typename TIn>
struct Ragged;

// In pieces of four; the row's last is read as the four values that end it.
template <>
struct Ragged<float> {
    f32x4 x[2];
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, int at, int c, int width, bool there) {
#pragma unroll
        for (int i = 0; i < 2; ++i, c += 4) {
            if (width >= 4) {
                const int off = there && c < width ? (at + min(c, width - 4)) * 4 : mfma::kOutside;
                x[i] = __builtin_bit_cast(f32x4, mfma::buf_load16<mfma::kPolicyDefault>(r, off));
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int off = there && c + e < width ? (at + c + e) * 4 : mfma::kOutside;
                    x[i][e] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0));
                }
            }
        }
    }
    __device__ __forceinline__ Eight<float> get(int, int c, int width) const {
        Eight<float> out;
#pragma unroll
        for (int i = 0; i < 2; ++i, c += 4) {
            f32x4 v = x[i];
            const int by = width >= 4 && c < width ? max(c + 4 - width, 0) : 0;
            if (by & 1) v = f32x4{v[1], v[2], v[3], 0.f};
            if (by & 2) v = f32x4{v[2], v[3], 0.f, 0.f};
            out.v[i] = __builtin_bit_cast(uint4, v);
        }
        return out;
    }
};

// Through the words they lie in.
template <>
struct Ragged<bf16_t> {
    uint32_t w[5];
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, int at, int c, int width, bool there) {
        const int odd = at & 1, n = there && width > c ? width - c : -5;
#pragma unroll
        for (int i = 0; i < 5; ++i)
            w[i] = __builtin_amdgcn_raw_buffer_load_b32(r, 2 * i - odd < n ? (at + c - odd + 2 * i) * 2 : mfma::kOutside, 0, 0);
    }
    __device__ __forceinline__ Eight<bf16_t> get(int at, int c, int width) const {
        Eight<bf16_t> out;
        uint32_t x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int n = width - c - 2 * i;
            x[i] = __builtin_amdgcn_alignbit(w[i + 1], w[i], 16 * (at & 1));
            x[i] = n > 1 ? x[i] : n > 0 ? x[i] & 0xffffu : 0u;
        }
        out.v[0] = make_uint4(x[0], x[1], x[2], x[3]);
        return out;
    }
};

// A view of `live` rows from p on for them, and the element of it that p is: from the
// word that p lies in (arrays start 16-byte aligned) to the end of the last one, whose
// other half, where it lies behind the array, shares its allocation and is cut off.
template <typename TIn>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t ragged_view(const TIn* p, int64_t stride, int live, int width, int& at) {
    at = int(reinterpret_cast<uintptr_t>(p) & 3) / int(sizeof(TIn));
    const int64_t bytes = ((live - 1) * stride + width + at) * int(sizeof(TIn));
    return mfma::make_rsrc(p - at, (bytes + 3) & ~int64_t(3));
}

// Byte offset of the 16-byte piece from column `col` of a row; outside every view past the row's width.
template <typename TIn>
__device__ __forceinline__ int piece_at(int row, int stride, int col, int width) {
    return col < width ? (row * stride + col) * int(sizeof(TIn)) : mfma::kOutside;
}

// 64 rows of K values: each thread's 8-value pieces in registers and then in a tile.
// Through a view that ends with the last live row: in 16-byte pieces (kVec), or
// value by value.
template <typename TIn, int K, int NT, bool kVec>
struct Stage {
    static constexpr int kPer = kChunk * (K / 8) / NT, kVecs = Eight<TIn>::kVecs;
    std::conditional_t<kVec, Eight<TIn>, Ragged<TIn>> x[kPer];
    int off[kVec ? kPer * kVecs : 1];
    int stride_, width_, at_;  // of the rows loaded
    // Wide rows compute the offsets of their values each time: kept, they take the registers that
    // the products need (32 streams of 3000 fp32 tokens, 100 x 127: the walk 216 -> 173 us; 96
    // of 1500 bf16 ones, 33 x 50: kept 120, again 132).
    static constexpr bool kAgain = K * sizeof(TIn) > 128;
    __device__ __forceinline__ void init(int64_t stride, int width) {
        stride_ = int(stride), width_ = width;
        if constexpr (kVec) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int q = int(threadIdx.x) + i * NT, row = q / (K / 8), u = q % (K / 8);
#pragma unroll
                for (int j = 0; j < kVecs; ++j) off[i * kVecs + j] = piece_at<TIn>(row, int(stride), 8 * u + 4 * j, width);
            }
        }
    }
    // Rows of p, `live` of them there.
    __device__ __forceinline__ void load(const TIn* p, int live) {
        if constexpr (kVec) {
            const auto r = mfma::make_rsrc(p, ((live - 1) * int64_t(stride_) + width_) * int(sizeof(TIn)));
#pragma unroll
            for (int i = 0; i < kPer; ++i)
#pragma unroll
                for (int j = 0; j < kVecs; ++j) x[i].v[j] = mfma::buf_load16<mfma::kPolicyDefault>(r, off[i * kVecs + j]);
        } else {
            const auto r = ragged_view(p, stride_, live, width_, at_);
            int tid = threadIdx.x;
            if constexpr (kAgain) asm volatile("" : "+v"(tid));
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int q = tid + i * NT, row = q / (K / 8), u = q % (K / 8);
                x[i].load(r, at_ + row * stride_, 8 * u, width_, row < live);
            }
        }
    }
    __device__ __forceinline__ void put(unsigned char* t) const {
        int tid = threadIdx.x;
        if constexpr (!kVec && kAgain) asm volatile("" : "+v"(tid));
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int q = tid + i * NT, row = q / (K / 8), u = q % (K / 8);
            Eight<TIn> e;
            if constexpr (kVec)
                e = x[i];
            else
                e = x[i].get(at_ + row * stride_, 8 * u, width_);
#pragma unroll
            for (int j = 0; j < kVecs; ++j) *reinterpret_cast<uint4*>(t + Tile<TIn, K>::at(row, kVecs * u + j)) = e.v[j];
        }
    }
};

// T or M of a chunk in memory: a lower triangle [64][64], as fp32 values or as three
// parts of bf16.  A part is rows 32 .. 63, then the first half of rows 0 .. 31: what
// is right of it is not read anywhere.  (Split where they are made, not in the walks,
// whose chains would wait for it: 128 streams of 4096 bf16 tokens, 128 x 128, solve and
// walks 104 + 437 + 405 -> 116 + 406 + 382 us.)
template <typename E>
struct SquareOf {
    static constexpr int64_t kBytes = kChunk * kChunk * 4;
    // Four (eight) values from column `col` of a row, their first `parts` parts.
    __device__ __forceinline__ static void put4(unsigned char* p, int row, int col, const f32x4& x, int) {
        *reinterpret_cast<f32x4*>(p + (row * kChunk + col) * 4) = x;
    }
    __device__ __forceinline__ static void put8(unsigned char* p, int row, int col, const f32x4& x, const f32x4& y) {
        put4(p, row, col, x, 1), put4(p, row, col + 4, y, 1);
    }
};
template <>
struct SquareOf<bf16_t> {
    static constexpr int kHalf = 32 * kChunk * 2, kPart = kHalf + kHalf / 2;
    static constexpr int64_t kBytes = 3 * kPart;
    __device__ __forceinline__ static int at(int row, int col) {
        return row < 32 ? kHalf + (row * 32 + col) * 2 : ((row - 32) * kChunk + col) * 2;
    }
    __device__ __forceinline__ static void put4(unsigned char* p, int row, int col, f32x4 x, int parts) {
        if (row < 32 && col >= 32) return;
        p += at(row, col);
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i < 2 || parts > 2) *reinterpret_cast<uint2*>(p + i * kPart) = take_part(x);
    }
    __device__ __forceinline__ static void put8(unsigned char* p, int row, int col, f32x4 x, f32x4 y) {
        if (row < 32 && col >= 32) return;
        p += at(row, col);
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            const uint2 a = take_part(x), b = take_part(y);
            *reinterpret_cast<uint4*>(p + i * kPart) = make_uint4(a.x, a.y, b.x, b.y);
        }
    }
};

// Its first P parts (or its values) to a tile in as many planes, by a walk's threads.
template <typename E, int P>
struct StageSquare {
    f32x4 x[4];
    __device__ __forceinline__ void load(const unsigned char* p) {
        const auto r = mfma::make_rsrc(p, SquareOf<E>::kBytes);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            x[i] = __builtin_bit_cast(f32x4, mfma::buf_load16<mfma::kPolicyDefault>(r, 16 * (int(threadIdx.x) + i * kThreads)));
    }
    __device__ __forceinline__ void put(unsigned char* t) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int q = int(threadIdx.x) + i * kThreads;
            *reinterpret_cast<f32x4*>(t + Tile<E, 64>::at(q / 16, q % 16)) = x[i];
        }
    }
};
template <int P>
struct StageSquare<bf16_t, P> {
    static_assert(kThreads == 256);
    using S = SquareOf<bf16_t>;
    using T = Tile<bf16_t, 64>;
    uint4 low[P], high[(P + 1) / 2];  // rows 32 .. 63, a part each; rows 0 .. 31, two parts each
    __device__ __forceinline__ void load(const unsigned char* p) {
        const int tid = threadIdx.x;
        const auto r = mfma::make_rsrc(p, P * S::kPart);
#pragma unroll
        for (int i = 0; i < P; ++i) low[i] = mfma::buf_load16<mfma::kPolicyDefault>(r, i * S::kPart + 16 * tid);
#pragma unroll
        for (int i = 0; i < (P + 1) / 2; ++i)  // past the last part, outside the view
            high[i] = mfma::buf_load16<mfma::kPolicyDefault>(r, (2 * i + (tid >> 7)) * S::kPart + S::kHalf + 16 * (tid & 127));
    }
    __device__ __forceinline__ void put(unsigned char* t) const {
        const int tid = threadIdx.x;
#pragma unroll
        for (int i = 0; i < P; ++i) *reinterpret_cast<uint4*>(t + i * T::kBytes + T::at(32 + (tid >> 3), tid & 7)) = low[i];
#pragma unroll
        for (int i = 0; i < (P + 1) / 2; ++i)
            if (2 * i + 1 < P || tid < 128)
                *reinterpret_cast<uint4*>(t + (2 * i + (tid >> 7)) * T::kBytes + T::at((tid & 127) >> 2, tid & 3)) = high[i];
    }
};

// ---- what the kernels share ----

constexpr double kLog2e = 1.4426950408889634074;

struct DeltaArgs {
    const void *q, *k, *v, *gate, *beta;
    const float* state;
    void* out;
    float* final_state;
    unsigned char *tm, *mm;  // [N][chunks] of T and M, as SquareOf has them
    float* vec;     // [N][chunks][128]: E, then Z b
    float *st, *yt;  // nullable: [N][chunks][dvp] columns of S [DK] and Y [64]
    // Segments of seg_chunks chunks that are walked at once, from starts [N][segs][dk][dv];
    // a segment takes a state s to map_a s + map_x, [N][segs][dk][dk] and [dk][dv].
    float *starts, *map_a, *map_x;
    int segs, seg_chunks;
    int64_t N, T;
    int64_t qn, qt, kn, kt, vn, vt;
    Live live;
    int group, dk, dv, dvp, chunks;  // group: value streams of a key stream
    int gate_f32, form;
    int vec_k, vec_v, vec_o;  // rows of q and k, of v, of out (and dout) in 16-byte pieces
    float scale;

    // Streams and their chunks have 32 bits: divisions of 64 take hundreds of instructions
    // before a workgroup's first load.
    __device__ __forceinline__ int64_t key_stream(int64_t n) const { return unsigned(n) / unsigned(group); }
    __device__ __forceinline__ int64_t len_of(int64_t n) const {
        if (!live.lengths) return T;
        const int64_t len = live.lengths[unsigned(n) / unsigned(live.group)];
        return len < 0 ? 0 : len < T ? len : T;
    }
};

// Log decays below this are taken as this: e^-200 is zero in 32 bits, and a sum
// of them still has digits for what follows.
constexpr float kLowestLog = -200.f;

__device__ __forceinline__ float gate_value(const void* p, int64_t i, int f32) {
    return f32 ? static_cast<const float*>(p)[i] : to_f32(static_cast<const bf16_t*>(p)[i]);
}
// In two steps, for a load that is on its way while other things go on.
__device__ __forceinline__ uint32_t gate_bits(const void* p, int64_t i, int f32) {
    return f32 ? static_cast<const uint32_t*>(p)[i] : static_cast<const uint16_t*>(p)[i];
}
__device__ __forceinline__ float gate_of(uint32_t bits, int f32) { return __uint_as_float(f32 ? bits : bits << 16); }
__device__ __forceinline__ float log_decay(float g, int form) {
    const float l = form == RACE_GATE_LOG ? g : fminf(g, 0.f) - log1pf(expf(-fabsf(g)));
    return l < kLowestLog ? kLowestLog : l;
}

// Four values to memory, next to each other.
__device__ __forceinline__ void store4_of(float* p, const f32x4& x) { *reinterpret_cast<f32x4*>(p) = x; }
__device__ __forceinline__ void store4_of(bf16_t* p, const f32x4& x) {
    *reinterpret_cast<uint2*>(p) = make_uint2(mfma::pack2(x[0], x[1]), mfma::pack2(x[2], x[3]));
}

// Values (row, col) of a state [dk][dv], zero outside, through a buffer that ends with
// it: a value chosen after its load would get a branch around the load and a wait
// behind it, 32 of them at the start of a walk.
struct StateView {
    __amdgpu_buffer_rsrc_t r;
    int dk, dv;
    __device__ __forceinline__ StateView(const float* s, int dk, int dv)
        : r(mfma::make_rsrc(s, int64_t(dk) * dv * 4)), dk(dk), dv(dv) {}
    __device__ __forceinline__ float one(int row, int col) const {
        const int off = row < dk && col < dv ? (row * dv + col) * 4 : mfma::kOutside;
        return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0));
    }
    __device__ __forceinline__ f32x4 four(int row, int col) const {  // dv a multiple of 4
        const int off = row < dk && col < dv ? (row * dv + col) * 4 : mfma::kOutside;
        return __builtin_bit_cast(f32x4, mfma::buf_load16<mfma::kPolicyDefault>(r, off));
    }
};

// Whether two workgroups that walk chunks share a CU, each with one buffer, as narrow
// keys' registers and tiles allow, and the maps' (no Q and M).  192 streams of 577
// bf16 tokens, 64 x 128: the walk 52 -> 44 us; beside outputs, keys of 128 leave no LDS
// for a second.
constexpr bool two_a_cu(int row_bytes, bool maps) { return row_bytes <= (maps ? 256 : 128); }

// A chunk's tiles in LDS (bytes from its buffer's start); T in three parts, M in MP.
template <typename TIn, int DK, int MP, bool kOutputs = true, bool kTwoBuffers = kOutputs>
struct ChunkLds {
    static constexpr int kK = 0, kT = Tile<TIn, DK>::kBytes, kV = kT + kPartsBytes<TIn, 64, 3>, kVec = kV + Tile<TIn, 64>::kBytes;
    static constexpr int kQ = kVec + 512, kM = kQ + Tile<TIn, DK>::kBytes;
    static constexpr int kBytes = kOutputs ? kM + kPartsBytes<TIn, 64, MP> : kQ;
    // Two buffers, where they leave the workgroup its LDS: one barrier a chunk.
    static constexpr int kBuffers = kTwoBuffers && kOutputs && 2 * kBytes <= kGfx950LdsBytes ? 2 : 1;
};

// Consecutive streams on different XCDs, a stream's column blocks on one (they
// read the same tiles): workgroups go to the XCDs in turn.
__device__ __forceinline__ bool stream_and_block(int64_t N, int blocks, int64_t& n, int& cb) {
    const int64_t id = blockIdx.x, eight = id / (8 * blocks);
    const int in = int(id - eight * 8 * blocks);
    n = eight * 8 + (in & 7), cb = in >> 3;
    return n < N;
}

// ---- the segments' starts ----

// starts[0] = the state, starts[p + 1] = map_a[p] starts[p] + map_x[p], the first
// segment's map_x being what follows it; backward (kBack) from the last segment on,
// with the maps transposed.  Products are fp32.  A workgroup has 16 columns
// and a wave a quarter of the rows, whose part of the maps it loads two segments ahead; the columns meet in LDS, two copies in turn.
template <int DK, bool kBack>
__global__ __launch_bounds__(kThreads) void delta_join_kernel(const DeltaArgs a) {
    constexpr int NI = DK / 64, NJ = DK / 16, kPitch = DK + 4;
    __shared__ __align__(16) float cols[2][16 * kPitch];
    const int64_t n = blockIdx.y;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, lr = lane & 15;
    const int col = blockIdx.x * 16 + lr, r0 = wave * (DK / 4);
    const bool whole = a.dk % 4 == 0;
    struct Maps {
        f32x4 X[NI], A[NI][NJ];  // rows r0 + 16 i + 4 g + r; rows r0 + 16 i + lr, columns 16 j + 4 g + r
    } even, odd;
    f32x4 S[NI];
    auto rows = [&](const float* p, f32x4 (&x)[NI]) {
        const StateView s(p, a.dk, a.dv);
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) x[i][r] = s.one(r0 + 16 * i + 4 * g + r, col);
    };
    auto load = [&](Maps& m, int p) {
        const int64_t at = n * a.segs + p;
        rows(a.map_x + at * a.dk * a.dv, m.X);
        const StateView from(a.map_a + at * a.dk * a.dk, a.dk, a.dk);
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int row = r0 + 16 * i + lr, c = 16 * j + 4 * g;
                if constexpr (kBack) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) m.A[i][j][r] = from.one(c + r, row);
                } else if (whole) {
                    m.A[i][j] = from.four(row, c);
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r) m.A[i][j][r] = from.one(row, c + r);
                }
            }
    };
    if (a.state) {
        rows(a.state + n * a.dk * a.dv, S);
    } else {
#pragma unroll
        for (int i = 0; i < NI; ++i) S[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    auto segment = [&](int step) { return kBack ? a.segs - 1 - step : step; };
    auto step = [&](int p, Maps& m) {
        float* to = a.starts + (n * a.segs + segment(p)) * a.dk * a.dv;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = r0 + 16 * i + 4 * g + r;
                if (col < a.dv && row < a.dk) to[row * a.dv + col] = S[i][r];
            }
        if (p + 1 == a.segs) return;
        if (p > 0) {
            float* c = cols[p & 1];
#pragma unroll
            for (int i = 0; i < NI; ++i) *reinterpret_cast<f32x4*>(c + lr * kPitch + r0 + 16 * i + 4 * g) = S[i];
            __syncthreads();
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const f32x4 s = *reinterpret_cast<const f32x4*>(c + lr * kPitch + 16 * j + 4 * g);
#pragma unroll
                for (int i = 0; i < NI; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) m.X[i] = mfma::mfma4(m.A[i][j][r], s[r], m.X[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) S[i] = m.X[i];
        if (p + 3 < a.segs) load(m, segment(p + 2));
    };
    rows(a.map_x + (n * a.segs + segment(0)) * a.dk * a.dv, even.X);
    if (a.segs > 2) load(odd, segment(1));
    for (int p = 0; p < a.segs; p += 2) {
        step(p, even);
        if (p + 1 < a.segs) step(p + 1, odd);
    }
}

// ---- host ----

inline int dk_padded(const DeltaRule& r) { return r.dk <= 64 ? 64 : 128; }

// Whether rows of this width and these strides are whole 16-byte pieces.  (That 64 of them
// lie within a view's 32-bit offsets is the API's limit on token strides, 2^22.)
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
    a.vec_o = whole_pieces(r, r.dv, {});
    a.scale = r.scale;
    return a;
}

template <int DK, bool kBack>
inline void launch_join(const DeltaRule& r, const DeltaArgs& a, hipStream_t stream) {
    delta_join_kernel<DK, kBack><<<dim3(unsigned(r.dv + 15) / 16, unsigned(r.N)), kThreads, 0, stream>>>(a);
}

inline int64_t round256(int64_t bytes) { return (bytes + 255) / 256 * 256; }

}  // namespace delta
}  // namespace race
