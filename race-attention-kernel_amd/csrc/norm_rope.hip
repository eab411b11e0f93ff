// norm_rope.hip -- every head's query and key rows normed and rotated, from a
// projection's [B][T][H][d] to the op's streams [B * H][T][d], in one pass:
//
//     n = x / sqrt(mean(x^2) + eps) * w           (over the d values of a row)
//     (y_i, y_j) = (n_i cos f - n_j sin f, n_i sin f + n_j cos f),  f = position * freq[p]
//
// for the first 2 P values of a row as P pairs (i, j) = (p, p + P), or (2p,
// 2p + 1); the others pass.  With several position axes (time, height, width)
// each takes a run of the pairs.  And its gradients, with g the rotation of the
// upstream row by -f, r the reciprocal root and u = x r:
//
//     dw = sum over rows of g u,   dx = r (g w - u mean(g w u)).
//
// Bound by memory: rows in and rows out once.  A workgroup takes a tile of
// tokens and a group of heads.  It issues the loads of its rows, then puts the
// tile's cosines and sines into LDS, each once for all heads: the angle is the
// product in 64 bits, in turns, less its whole turns, so that far positions
// keep their digits.  A lane then holds V pairs of a row, both halves, and a
// row's sums run over its few lanes.  Consecutive row slots are consecutive
// tokens of one head, so a head's part of the tile leaves as one run.
// The weights' gradients are summed per lane, then per workgroup through LDS,
// then over the workgroups by a second kernel, all in a fixed order.
#include <algorithm>

#include "row_run.h"

namespace race {
namespace {

// Queries (0) and keys (1) of a launch.
struct RopeTensor {
    const void* x;
    const void* w;      // nullable: ones
    void* out;          // forward: the streams; backward: dx, nullable
    const void* up;     // backward: the upstream streams
    int64_t xb, xt, xh; // strides of x
    int heads, group, groups;  // heads of a workgroup, and workgroups a token tile takes
    int tile_shift;            // tokens of a workgroup's tile, as a power of two
};

struct RopeArgs {
    RopeTensor t[2];
    const void* pos;
    const float* freq;
    float* partial;  // backward: [groups of both][gridDim.x][d], nullable
    int64_t pa, pb, pt;
    int T, tokens, d, pairs;
    int ends[3];  // first pair of axes 1 .. 3
    int lane_shift;  // lanes of a row, as a power of two
    int pos64, norm, w_f32;
    float eps;
};

// Weights c .. c + V - 1 (ones without any), zeros where `in` is false.
template <int V>
__device__ __forceinline__ void load_weights(float (&x)[V], const RopeTensor& t, int w_f32, int c, bool in) {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = in ? 1.f : 0.f;
    if (!t.w || !in) return;
    if (w_f32) {
        constexpr int kPer = V >= 4 ? 4 : 1;
#pragma unroll
        for (int i = 0; i < V; i += kPer) {
            Run<float, kPer> r;
            r.load(static_cast<const float*>(t.w) + c + i);
#pragma unroll
            for (int j = 0; j < kPer; ++j) x[i + j] = r.get(j);
        }
    } else {
        Run<bf16_t, V> r;
        r.load(static_cast<const bf16_t*>(t.w) + c);
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = r.get(i);
    }
}

// Floats of one token's cosines and sines; the four more spread the tokens'
// reads over the banks.
__host__ __device__ inline int table_pitch(int pairs) { return 2 * ((pairs + 3) & ~3) + 4; }

// Cosines (row start) and sines (half a row on) of the tile's tokens.
__device__ __forceinline__ void fill_table(float* table, const RopeArgs& a, int first, int tile) {
    const int pitch = table_pitch(a.pairs), half = (a.pairs + 3) & ~3;
    for (int e = threadIdx.x; e < tile * a.pairs; e += kThreads) {
        const int tok = e / a.pairs, p = e - tok * a.pairs, i = first + tok;
        if (i >= a.tokens) break;
        const int b = i / a.T, t = i - b * a.T;
        const int axis = (p >= a.ends[0]) + (p >= a.ends[1]) + (p >= a.ends[2]);
        const int64_t at = axis * a.pa + b * a.pb + t * a.pt;
        const double pos = a.pos64 ? double(static_cast<const int64_t*>(a.pos)[at])
                                   : double(static_cast<const int32_t*>(a.pos)[at]);
        const double turns = pos * (double(a.freq[p]) * 0.15915494309189533577);  // 1 / (2 pi)
        float s, c;
        sincospif(2.f * float(turns - rint(turns)), &s, &c);
        table[tok * pitch + p] = c;
        table[tok * pitch + half + p] = s;
    }
}

// What a lane holds of a row: NS slots of V pairs (values o1 .. and o2 ..).
template <int V, int NS, bool kInterleaved>
struct Lanes {
    int pair[NS], o1[NS], o2[NS];
    bool one[NS], two[NS];  // the slot's first and second values are there
    __device__ __forceinline__ Lanes(const RopeArgs& a, int l) {
        const int slots = (a.d + 1) / 2;  // pairs, turned or not; an odd width leaves one half empty
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            const int p = ((j << a.lane_shift) + l) * V;
            pair[j] = p;
            if constexpr (kInterleaved) {
                o1[j] = 2 * p;
                o2[j] = V == 1 ? 2 * p + 1 : 2 * p + V;
            } else {
                o1[j] = p < a.pairs ? p : a.pairs + p;
                o2[j] = p < a.pairs ? p + a.pairs : p + slots;
            }
            one[j] = p < slots;
            two[j] = one[j] && o2[j] < a.d;
        }
    }
};

// Values (a, b) of a slot as its pairs' firsts and seconds, and back.
template <int V, bool kInterleaved>
__device__ __forceinline__ void to_pairs(float (&a)[V], float (&b)[V]) {
    if constexpr (kInterleaved && V > 1) {
        float f[V], s[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            f[i] = 2 * i < V ? a[2 * i] : b[2 * i - V];
            s[i] = 2 * i < V ? a[2 * i + 1] : b[2 * i + 1 - V];
        }
#pragma unroll
        for (int i = 0; i < V; ++i) a[i] = f[i], b[i] = s[i];
    }
}
template <int V, bool kInterleaved>
__device__ __forceinline__ void from_pairs(float (&a)[V], float (&b)[V]) {
    if constexpr (kInterleaved && V > 1) {
        float x[2 * V];
#pragma unroll
        for (int i = 0; i < V; ++i) x[2 * i] = a[i], x[2 * i + 1] = b[i];
#pragma unroll
        for (int i = 0; i < V; ++i) a[i] = x[i], b[i] = x[V + i];
    }
}

// Turns the slot's pairs by the table's angles (kBack: the other way).
template <int V, bool kBack>
__device__ __forceinline__ void rotate(const float* row, int half, int pair, int pairs, float (&x)[V], float (&y)[V]) {
    if (pair >= pairs) return;
    float c[V], s[V];
    if constexpr (V >= 4) {
        // The rows are padded to whole fours; pairs past the last are not turned.
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            if (pair + i < pairs) {
                const float4 cv = *reinterpret_cast<const float4*>(row + pair + i);
                const float4 sv = *reinterpret_cast<const float4*>(row + half + pair + i);
                c[i] = cv.x, c[i + 1] = cv.y, c[i + 2] = cv.z, c[i + 3] = cv.w;
                s[i] = sv.x, s[i + 1] = sv.y, s[i + 2] = sv.z, s[i + 3] = sv.w;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) c[i] = row[pair + i], s[i] = row[half + pair + i];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const bool in = pair + i < pairs;
        const float ci = in ? c[i] : 1.f, si = in ? (kBack ? -s[i] : s[i]) : 0.f;
        const float a = x[i], b = y[i];
        x[i] = a * ci - b * si;
        y[i] = a * si + b * ci;
    }
}

__device__ __forceinline__ float over_row(float x, int lane_shift) {
    for (int k = 0; k < lane_shift; ++k) x += __shfl_xor(x, 1 << k);
    return x;
}

// The workgroup's tensor and first head.
__device__ __forceinline__ int head_group(const RopeArgs& a, int& h0) {
    const int z = int(blockIdx.y) < a.t[0].groups ? 0 : 1;
    h0 = (int(blockIdx.y) - (z ? a.t[0].groups : 0)) * a.t[z].group;
    return z;
}

// blockIdx.x takes every gridDim.x-th token tile, blockIdx.y is a head group;
// NR rows per lane group.
template <typename TIn, int V, int NS, int NR, bool kInterleaved>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(const RopeArgs a) {
    extern __shared__ __align__(16) float table[];
    using X = Run<TIn, V>;
    int h0;
    const int z = head_group(a, h0);
    const RopeTensor t = z ? a.t[1] : a.t[0];
    const int tile = 1 << t.tile_shift, tiles = (a.tokens + tile - 1) >> t.tile_shift;
    const int l = threadIdx.x & ((1 << a.lane_shift) - 1), r0 = threadIdx.x >> a.lane_shift;
    const int row_step = kThreads >> a.lane_shift;
    const int heads = min(t.group, t.heads - h0);
    const int pitch = table_pitch(a.pairs), half = (a.pairs + 3) & ~3;
    const Lanes<V, NS, kInterleaved> ln(a, l);
    float w1[NS][V], w2[NS][V];
#pragma unroll
    for (int j = 0; j < NS; ++j) {
        load_weights<V>(w1[j], t, a.w_f32, ln.o1[j], ln.one[j]);
        load_weights<V>(w2[j], t, a.w_f32, ln.o2[j], ln.two[j]);
    }
    for (int ti = blockIdx.x; ti < tiles; ti += gridDim.x) {
        const int first = ti << t.tile_shift;
        X x1[NR][NS], x2[NR][NS];
        int64_t to[NR];
        bool there[NR];
#pragma unroll
        for (int k = 0; k < NR; ++k) {
            const int row = r0 + k * row_step, i = first + (row & (tile - 1)), hl = row >> t.tile_shift;
            there[k] = hl < heads && i < a.tokens;
            const int b = i / a.T, tt = i - b * a.T, h = h0 + hl;
            const TIn* p = static_cast<const TIn*>(t.x) + b * t.xb + tt * t.xt + h * t.xh;
            to[k] = ((int64_t(b) * t.heads + h) * a.T + tt) * a.d;
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                x1[k][j].clear(), x2[k][j].clear();
                if (there[k] && ln.one[j]) x1[k][j].load(p + ln.o1[j]);
                if (there[k] && ln.two[j]) x2[k][j].load(p + ln.o2[j]);
            }
        }
        if (ti != int(blockIdx.x)) __syncthreads();  // the tile before is done with the table
        fill_table(table, a, first, tile);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NR; ++k) {
            float y1[NS][V], y2[NS][V], ss = 0.f;
#pragma unroll
            for (int j = 0; j < NS; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    y1[j][i] = x1[k][j].get(i), y2[j][i] = x2[k][j].get(i);
                    ss = fmaf(y1[j][i], y1[j][i], fmaf(y2[j][i], y2[j][i], ss));
                }
            if (a.norm) {
                const float r = rsqrtf(over_row(ss, a.lane_shift) / float(a.d) + a.eps);
#pragma unroll
                for (int j = 0; j < NS; ++j)
#pragma unroll
                    for (int i = 0; i < V; ++i) y1[j][i] *= r * w1[j][i], y2[j][i] *= r * w2[j][i];
            }
            if (!there[k]) continue;
            const float* row = table + ((r0 + k * row_step) & (tile - 1)) * pitch;
            TIn* o = static_cast<TIn*>(t.out) + to[k];
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                to_pairs<V, kInterleaved>(y1[j], y2[j]);
                rotate<V, false>(row, half, ln.pair[j], a.pairs, y1[j], y2[j]);
                from_pairs<V, kInterleaved>(y1[j], y2[j]);
                if (ln.one[j]) X::store(o + ln.o1[j], y1[j]);
                if (ln.two[j]) X::store(o + ln.o2[j], y2[j]);
            }
        }
    }
}

template <typename TIn, int V, int NS, int NR, bool kInterleaved>
__global__ __launch_bounds__(kThreads) void norm_rope_bwd_kernel(const RopeArgs a) {
    extern __shared__ __align__(16) float table[];
    using X = Run<TIn, V>;
    int h0;
    const int z = head_group(a, h0);
    const RopeTensor t = z ? a.t[1] : a.t[0];
    const int tile = 1 << t.tile_shift, tiles = (a.tokens + tile - 1) >> t.tile_shift;
    const int l = threadIdx.x & ((1 << a.lane_shift) - 1), r0 = threadIdx.x >> a.lane_shift;
    const int row_step = kThreads >> a.lane_shift;
    const int heads = min(t.group, t.heads - h0);
    const int pitch = table_pitch(a.pairs), half = (a.pairs + 3) & ~3;
    const Lanes<V, NS, kInterleaved> ln(a, l);
    float w1[NS][V], w2[NS][V], dw1[NS][V], dw2[NS][V];
#pragma unroll
    for (int j = 0; j < NS; ++j) {
        load_weights<V>(w1[j], t, a.w_f32, ln.o1[j], ln.one[j]);
        load_weights<V>(w2[j], t, a.w_f32, ln.o2[j], ln.two[j]);
#pragma unroll
        for (int i = 0; i < V; ++i) dw1[j][i] = dw2[j][i] = 0.f;
    }
    for (int ti = blockIdx.x; ti < tiles; ti += gridDim.x) {
        const int first = ti << t.tile_shift;
        X x1[NR][NS], x2[NR][NS], u1[NR][NS], u2[NR][NS];
        int64_t to[NR];
        bool there[NR];
#pragma unroll
        for (int k = 0; k < NR; ++k) {
            const int row = r0 + k * row_step, i = first + (row & (tile - 1)), hl = row >> t.tile_shift;
            there[k] = hl < heads && i < a.tokens;
            const int b = i / a.T, tt = i - b * a.T, h = h0 + hl;
            const TIn* p = static_cast<const TIn*>(t.x) + b * t.xb + tt * t.xt + h * t.xh;
            const TIn* up = static_cast<const TIn*>(t.up) + ((int64_t(b) * t.heads + h) * a.T + tt) * a.d;
            to[k] = (int64_t(i) * t.heads + h) * a.d;
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                x1[k][j].clear(), x2[k][j].clear(), u1[k][j].clear(), u2[k][j].clear();
                const bool one = there[k] && ln.one[j], two = there[k] && ln.two[j];
                if (one) u1[k][j].load(up + ln.o1[j]);
                if (two) u2[k][j].load(up + ln.o2[j]);
                if (a.norm && one) x1[k][j].load(p + ln.o1[j]);
                if (a.norm && two) x2[k][j].load(p + ln.o2[j]);
            }
        }
        if (ti != int(blockIdx.x)) __syncthreads();
        fill_table(table, a, first, tile);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NR; ++k) {
            const float* row = table + ((r0 + k * row_step) & (tile - 1)) * pitch;
            float g1[NS][V], g2[NS][V], ss = 0.f, gx = 0.f;
#pragma unroll
            for (int j = 0; j < NS; ++j) {
#pragma unroll
                for (int i = 0; i < V; ++i) g1[j][i] = u1[k][j].get(i), g2[j][i] = u2[k][j].get(i);
                if (there[k]) {
                    to_pairs<V, kInterleaved>(g1[j], g2[j]);
                    rotate<V, true>(row, half, ln.pair[j], a.pairs, g1[j], g2[j]);
                    from_pairs<V, kInterleaved>(g1[j], g2[j]);
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float xa = x1[k][j].get(i), xb = x2[k][j].get(i);
                    ss = fmaf(xa, xa, fmaf(xb, xb, ss));
                    gx = fmaf(g1[j][i] * w1[j][i], xa, fmaf(g2[j][i] * w2[j][i], xb, gx));
                }
            }
            if (a.norm) {
                // u = x r: dx = r (g w) - x (r^3 sum(g w x) / d).
                const float inv_d = 1.f / float(a.d);
                const float r = rsqrtf(over_row(ss, a.lane_shift) * inv_d + a.eps);
                const float m = over_row(gx, a.lane_shift) * inv_d * r * r * r;
#pragma unroll
                for (int j = 0; j < NS; ++j)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float xa = x1[k][j].get(i), xb = x2[k][j].get(i);
                        if (there[k]) {
                            dw1[j][i] = fmaf(g1[j][i], xa * r, dw1[j][i]);
                            dw2[j][i] = fmaf(g2[j][i], xb * r, dw2[j][i]);
                        }
                        g1[j][i] = fmaf(g1[j][i] * w1[j][i], r, -xa * m);
                        g2[j][i] = fmaf(g2[j][i] * w2[j][i], r, -xb * m);
                    }
            }
            if (!there[k] || !t.out) continue;
            TIn* o = static_cast<TIn*>(t.out) + to[k];
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                if (ln.one[j]) X::store(o + ln.o1[j], g1[j]);
                if (ln.two[j]) X::store(o + ln.o2[j], g2[j]);
            }
        }
    }
    if (!a.partial) return;
    // The row groups' sums, in order.
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NS; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (ln.one[j]) table[r0 * a.d + ln.o1[j] + i] = dw1[j][i];
            if (ln.two[j]) table[r0 * a.d + ln.o2[j] + i] = dw2[j][i];
        }
    __syncthreads();
    for (int c = threadIdx.x; c < a.d; c += kThreads) {
        float s = 0.f;
        for (int r = 0; r < row_step; ++r) s += table[r * a.d + c];
        a.partial[(int64_t(blockIdx.y) * gridDim.x + blockIdx.x) * a.d + c] = s;
    }
}

// dw[c] = the sum of the partial rows of one tensor: 32 columns and 32 runs of
// rows a workgroup; blockIdx.y is the tensor.
struct RopeSums {
    const float* partial;
    void* dw[2];
    int rows[2];  // partial rows of the queries, then the keys
    int d, w_f32;
};
__global__ __launch_bounds__(1024) void rope_weight_sums_kernel(const RopeSums a) {
    const int z = blockIdx.y;
    column_sums(a.partial + int64_t(z ? a.rows[0] : 0) * a.d, z ? a.rows[1] : a.rows[0], a.d, z ? a.dw[1] : a.dw[0], a.w_f32);
}

int log2_up(int64_t x) {
    int k = 0;
    while ((int64_t(1) << k) < x) ++k;
    return k;
}

// Values per 16- or 8-byte piece that every offset, stride and pair run of the
// call is a multiple of; 1 for any others.
int rope_vector(const NormRope& r) {
    auto whole = [&](int v) {
        if (r.d % (2 * v) != 0 || (!r.interleaved && r.pairs % v != 0)) return false;
        for (int z = 0; z < 2; ++z) {
            if (r.heads[z] == 0) continue;
            for (int64_t s : {r.xb[z], r.xt[z], r.xh[z]})
                if (s % v != 0) return false;
        }
        return true;
    };
    if (r.dtype == RACE_BF16 && whole(8)) return 8;
    return whole(4) ? 4 : 1;
}

// A launch: rows per workgroup, the tensors' tiles and head groups.
struct RopePlan {
    RopeArgs a;
    dim3 grid;
    size_t lds;
    int rows_each;  // NR
};

// A lane group takes two rows where that leaves kRopeEnough workgroups (of 1 x
// 16384 tokens of 32 + 8 heads of 128 in bf16, forward: 69 us; one row 123, four
// rows 77, whose registers leave fewer waves).  The workgroups stay for several
// tiles: 2560 forward (69 us; one tile each 75), and backward two rounds of what
// is resident (bf16 two rounds of three per CU: 8 x 8192 tokens of 16 + 16 heads
// of 64 165 us, 1280 workgroups 179, 2048 178; fp32 one of four: 32 x 1024 tokens
// of 12 + 12 heads of 64 119 us, 1536 workgroups 138).
constexpr int kRopeEnough = 512, kRopeFwdWorkgroups = 2560, kRopeBwdWorkgroups = 1536, kRopeBwdWorkgroupsF32 = 1024;
constexpr int kRopeTableBytes = 64 * 1024;

RopePlan rope_plan(const NormRope& r, const void* const (&x)[2], const void* const (&w)[2], bool backward) {
    RopePlan p = {};
    RopeArgs& a = p.a;
    const int v = rope_vector(r), slots = (r.d + 1) / 2;
    a.T = int(r.T), a.tokens = int(r.B * r.T), a.d = r.d, a.pairs = r.pairs;
    a.pos = r.positions, a.freq = r.inv_freq;
    a.pa = r.pa, a.pb = r.pb, a.pt = r.pt, a.pos64 = r.pos64;
    for (int i = 0, e = 0; i < 3; ++i) a.ends[i] = e = i + 1 < r.axes ? e + r.sections[i] : INT32_MAX;
    a.norm = r.norm, a.eps = r.eps, a.w_f32 = r.weight_dtype == RACE_F32;
    a.lane_shift = v == 1 ? 5 : log2_up((slots + v - 1) / v);
    const int lane_groups = kThreads >> a.lane_shift;
    const int64_t rows = int64_t(a.tokens) * (r.heads[0] + r.heads[1]);
    p.rows_each = v > 1 && rows >= int64_t(2) * lane_groups * kRopeEnough ? 2 : 1;
    const int wg_rows = lane_groups * p.rows_each;
    int64_t most_tiles = 0;
    int groups = 0, tile_tokens = 0;
    for (int z = 0; z < 2; ++z) {
        RopeTensor& t = a.t[z];
        t.x = x[z], t.w = w[z];
        t.xb = r.xb[z], t.xt = r.xt[z], t.xh = r.xh[z];
        t.heads = r.heads[z];
        if (t.heads == 0 || !x[z]) {
            t.heads = 0, t.group = 1, t.groups = 0, t.tile_shift = 0;
            continue;
        }
        t.tile_shift = std::min({log2_up((wg_rows + t.heads - 1) / t.heads), log2_up(wg_rows), log2_up(a.tokens)});
        while ((int64_t(table_pitch(r.pairs)) * 4 << t.tile_shift) > kRopeTableBytes) --t.tile_shift;
        const int most = wg_rows >> t.tile_shift;
        t.groups = (t.heads + most - 1) / most;
        t.group = (t.heads + t.groups - 1) / t.groups;
        groups += t.groups;
        tile_tokens = std::max(tile_tokens, 1 << t.tile_shift);
        most_tiles = std::max<int64_t>(most_tiles, (a.tokens + (1 << t.tile_shift) - 1) >> t.tile_shift);
    }
    // The backward's workgroups leave one partial row each of the weights' gradients.
    const int wgs = !backward ? kRopeFwdWorkgroups : r.dtype == RACE_BF16 ? kRopeBwdWorkgroups : kRopeBwdWorkgroupsF32;
    p.grid = dim3(unsigned(std::min<int64_t>(most_tiles, std::max(1, wgs / std::max(groups, 1)))), unsigned(groups));
    p.lds = sizeof(float) * std::max<int64_t>(int64_t(tile_tokens) * table_pitch(r.pairs),
                                              backward ? int64_t(lane_groups) * r.d : 4);
    return p;
}

template <typename TIn, int V, int NS, int NR, bool kInterleaved>
void launch_rope(const RopePlan& p, bool backward, hipStream_t stream) {
    if (backward)
        norm_rope_bwd_kernel<TIn, V, NS, NR, kInterleaved><<<p.grid, kThreads, p.lds, stream>>>(p.a);
    else
        norm_rope_kernel<TIn, V, NS, NR, kInterleaved><<<p.grid, kThreads, p.lds, stream>>>(p.a);
}

template <typename TIn, int V, int NS>
void launch_rope_v(const NormRope& r, const RopePlan& p, bool backward, hipStream_t stream) {
    if constexpr (V > 1) {
        if (p.rows_each == 2) {
            if (r.interleaved) return launch_rope<TIn, V, NS, 2, true>(p, backward, stream);
            return launch_rope<TIn, V, NS, 2, false>(p, backward, stream);
        }
    }
    if (r.interleaved) return launch_rope<TIn, V, NS, 1, true>(p, backward, stream);
    return launch_rope<TIn, V, NS, 1, false>(p, backward, stream);
}

hipError_t launch_plan(const NormRope& r, const RopePlan& p, bool backward, hipStream_t stream) {
    // Slots of a lane: one, or up to four where pairs go one by one (32 lanes, d <= 256).
    const int v = rope_vector(r);
    if (r.dtype == RACE_BF16) {
        if (v == 8)
            launch_rope_v<bf16_t, 8, 1>(r, p, backward, stream);
        else if (v == 4)
            launch_rope_v<bf16_t, 4, 1>(r, p, backward, stream);
        else
            launch_rope_v<bf16_t, 1, 4>(r, p, backward, stream);
    } else if (v == 4) {
        launch_rope_v<float, 4, 1>(r, p, backward, stream);
    } else {
        launch_rope_v<float, 1, 4>(r, p, backward, stream);
    }
    return hipGetLastError();
}

}  // namespace

int64_t norm_rope_partial_floats(const NormRope& r) {
    return std::max<int64_t>(kRopeBwdWorkgroups, r.heads[0] + r.heads[1]) * r.d;
}

hipError_t launch_norm_rope(const NormRope& r, const void* const (&x)[2], const void* const (&w)[2], void* const (&out)[2],
                            hipStream_t stream) {
    RopePlan p = rope_plan(r, x, w, false);
    for (int z = 0; z < 2; ++z) p.a.t[z].out = out[z];
    return launch_plan(r, p, false, stream);
}

hipError_t launch_norm_rope_bwd(const NormRope& r, const void* const (&x)[2], const void* const (&w)[2],
                                const void* const (&up)[2], void* const (&dx)[2], void* const (&dw)[2], float* partial,
                                hipStream_t stream) {
    RopePlan p = rope_plan(r, x, w, true);
    for (int z = 0; z < 2; ++z) p.a.t[z].out = dx[z], p.a.t[z].up = up[z];
    const bool sums = dw[0] || dw[1];
    p.a.partial = sums ? partial : nullptr;
    const hipError_t err = launch_plan(r, p, true, stream);
    if (err != hipSuccess || !sums) return err;
    RopeSums s = {partial, {dw[0], dw[1]}, {}, r.d, p.a.w_f32};
    for (int z = 0; z < 2; ++z) s.rows[z] = p.a.t[z].groups * int(p.grid.x);
    rope_weight_sums_kernel<<<dim3(unsigned((r.d + 31) / 32), 2), 1024, 0, stream>>>(s);
    return hipGetLastError();
}

}  // namespace race
