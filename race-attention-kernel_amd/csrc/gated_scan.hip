// gated_scan.hip -- the gated linear recurrence and its gradients:
//
//     h_t = a_t h_{t-1} + u_t        per stream and channel, t = 0 .. T-1
//     a_t = sigmoid(g_t) or exp(g_t),  u_t = x_t or (1 - a_t) x_t
//
// from a carried state h_{-1} to the state after the last token, and with
// lambda_t = dh_t + mu_{t+1}, mu_t = a_t lambda_t (mu_T the gradient of the
// final state):
//
//     dx_t = lambda_t (or (1 - a_t) lambda_t),  dh_{-1} = mu_0,
//     dlog a_t = mu_t (h_{t-1} - (0 or x_t)),   dg_t = dlog a_t (1 - a_t or 1).
//
// mu runs backward through the same recurrence as h runs forward (mu_t = a_t
// mu_{t+1} + a_t dh_t), so both directions are one scan over pairs (P, H): a
// run of tokens takes a state s to P s + H.
//
// Bound by memory: x, g in and h out once, about 20 vector instructions an
// element.  A workgroup takes a block of channels (128 bytes of a row) of one
// stream through all its tokens, a tile of kTile tokens at a time: a thread
// has kRun consecutive tokens of V channels in registers (the next tile's rows
// loaded meanwhile), the threads' pairs are scanned over a wave by lane
// shuffles and over the waves through LDS, and every element is read once.  The
// state a tile starts from stays in 32 bits; with a gradient to come it is kept
// (one value per tile and channel), and the backward recomputes h from it
// exactly instead of from the rounded output.
// Few channels and many tokens are split over the tokens: one launch gives
// every segment's pair, the next starts each segment from the pairs before it.
// (A workgroup per tile that waits for the states of the tiles before it, which
// reads the rows once, took longer: 8 x 65536 x 64 bf16 107 us forward and 187
// backward against 82 and 120, 1 x 2^20 x 16 616 against 126: a state took 10 us
// to reach the workgroups of the next 64 tiles.)
// Sums have a fixed order: results are bitwise reproducible.
#include <algorithm>

#include "mfma_common.h"

namespace race {
namespace {

// V consecutive channels of a row, at a byte offset of a buffer.
template <typename TIn, int V>
struct Piece {
    static constexpr int kBytes = V * int(sizeof(TIn));
    using Raw = std::conditional_t<V == 1, TIn, std::conditional_t<sizeof(TIn) == 4, mfma::u32x4, mfma::u32x2>>;
    Raw v;
    template <int P>
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, int off) {
        if constexpr (kBytes == 16)
            v = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, P);
        else if constexpr (kBytes == 8)
            v = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, P);
        else if constexpr (kBytes == 4)
            v = __builtin_bit_cast(Raw, __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, P));
        else
            v = __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, P);
    }
    __device__ __forceinline__ float get(int j) const {
        if constexpr (V == 1)
            return to_f32(v);
        else if constexpr (sizeof(TIn) == 4)
            return __uint_as_float(v[j]);
        else
            return (j & 1) ? mfma::hi_half(v[j >> 1]) : mfma::lo_half(v[j >> 1]);
    }
    template <int P>
    __device__ __forceinline__ static void store(__amdgpu_buffer_rsrc_t r, int off, const float (&x)[V]) {
        if constexpr (kBytes == 16)
            __builtin_amdgcn_raw_buffer_store_b128(mfma::u32x4{__float_as_uint(x[0]), __float_as_uint(x[1]),
                                                               __float_as_uint(x[2]), __float_as_uint(x[3])},
                                                   r, off, 0, P);
        else if constexpr (kBytes == 8)
            __builtin_amdgcn_raw_buffer_store_b64(mfma::u32x2{mfma::pack2(x[0], x[1]), mfma::pack2(x[2], x[3])}, r, off,
                                                  0, P);
        else if constexpr (kBytes == 4)
            __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(x[0]), r, off, 0, P);
        else
            __builtin_amdgcn_raw_buffer_store_b16(f32_to_bf16(x[0]), r, off, 0, P);
    }
    __device__ __forceinline__ static void put(TIn* p, const float (&x)[V]) {
        if constexpr (V == 1)
            store_val(p, x[0]);
        else if constexpr (sizeof(TIn) == 4)
            *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
        else
            *reinterpret_cast<uint2*>(p) = make_uint2(mfma::pack2(x[0], x[1]), mfma::pack2(x[2], x[3]));
    }
};

// Where a thread past the channels reads: behind every tile's view, and with the
// steps over a thread's rows added still within 32 bits (ScanTile checks both).
constexpr int kPastTile = 1 << 30;

// The rows from `r0` on (at most kTile of them, before `end`) of an array with
// rows of D values `stride` apart: loads past them give zero, stores past them
// are dropped.
template <int kTile, typename T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_view(T* base, int64_t r0, int64_t end, int64_t stride, int64_t D) {
    const int64_t rows = min<int64_t>(end - r0, kTile);
    return mfma::make_rsrc(base + r0 * stride, rows > 0 ? ((rows - 1) * stride + D) * int64_t(sizeof(T)) : 0);
}

template <int V>
__device__ __forceinline__ void load_floats(float (&x)[V], const float* p) {
    if constexpr (V == 4) {
        const float4 f = *reinterpret_cast<const float4*>(p);
        x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = p[j];
    }
}
template <int V>
__device__ __forceinline__ void store_floats(float* p, const float (&x)[V]) {
    if constexpr (V == 4)
        *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    else
#pragma unroll
        for (int j = 0; j < V; ++j) p[j] = x[j];
}

// a and b = 1 - a of a gate value, each to its own last bits (b would lose
// them as a difference where a is near 1).  With t = exp(-|g|), sigmoid(|g|) =
// 1 / (1 + t) and sigmoid(-|g|) = t / (1 + t); t as 2^p with the rounding of
// p = -|g| log2(e) put back to first order.
template <int kForm>
__device__ __forceinline__ void open_gate(float g, float& a, float& b) {
    if constexpr (kForm == RACE_GATE_SIGMOID) {
        constexpr float kLog2e = 1.44269504f, kLog2eLo = 1.92596299e-8f, kLn2 = 0.693147181f;
        float x = -fabsf(g);
        x = x < -150.f ? -150.f : x;  // 0 from here on; NaN stays NaN
        const float p = x * kLog2e;
        const float e = fmaf(x, kLog2eLo, fmaf(x, kLog2e, -p));
        float t = __builtin_amdgcn_exp2f(p);
        t = fmaf(t, e * kLn2, t);
        const float r = __builtin_amdgcn_rcpf(1.f + t), tr = t * r;
        a = g >= 0.f ? r : tr;
        b = g >= 0.f ? tr : r;
    } else {
        a = expf(g);
        b = -expm1f(g);  // only where it is used
    }
}

struct ScanGeo {
    int64_t T, D;
    int64_t xn, xt, gn, gt;  // strides of x and the gates, in elements
    Live live;
    int64_t seg_len;  // tokens per segment, whole tiles
    int segs;
    int64_t tiles;    // records of a stream
};

struct ScanFwdArgs {
    const void *x, *gate;
    const float* state_in;  // nullable: zero
    void* out;
    float* state_out;  // nullable
    float* records;    // nullable: [N][tiles][D], the state each backward tile starts from
    float* pairs;      // [N][segs][2][D] with more than one segment
};

struct ScanBwdArgs {
    const void *x, *gate, *dout;
    const float* records;
    const float* dfinal;  // nullable: zero
    void *dx, *dgate;     // nullable
    float* dstate;        // nullable
    float* pairs;
};

// One workgroup's shape: CL lanes across channels, the others across tokens.
template <int NT, int CL, int R, int V>
struct ScanTile {
    static constexpr int kWaves = NT / 64, kTokenLanes = NT / CL, kTile = kTokenLanes * R, kChannels = CL * V;
    static constexpr int kLdsFloats = 2 * 2 * kWaves * kChannels;  // two buffers of the waves' pairs
    static constexpr int64_t kRowBytes = int64_t(RACE_SCAN_MAX_TOKEN_STRIDE) * 4;  // at most, from row to row
    static_assert((kTile - 1) * kRowBytes + int64_t(kScanMaxChannels) * 4 <= kPastTile, "behind the longest tile");
    static_assert(kPastTile + R * kRowBytes <= INT32_MAX, "offsets of 32 bits");
    // The threads' pairs (P, H), in token order for kUp and against it
    // otherwise, applied to `carry`: start = the state this thread's tokens begin
    // with, carry = the state after all of them; with kProduct, `product` takes
    // the product of every P too.  `lds` is one of the two buffers, in turn.
    template <bool kUp, bool kProduct>
    __device__ __forceinline__ static void join(float (&P)[V], float (&H)[V], float (&carry)[V], float (&start)[V],
                                                float (&product)[V], float* lds) {
        const int lane = threadIdx.x & 63, cl = lane % CL;
        const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
        for (int off = CL; off < 64; off *= 2) {
            const bool has = kUp ? lane >= off : lane + off < 64;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float p = kUp ? __shfl_up(P[j], off) : __shfl_down(P[j], off);
                const float h = kUp ? __shfl_up(H[j], off) : __shfl_down(H[j], off);
                if (has) {
                    H[j] = fmaf(P[j], h, H[j]);
                    P[j] *= p;
                }
            }
        }
        float* lp = lds;                        // [waves][channels]
        float* lh = lds + kWaves * kChannels;
        if (kUp ? lane >= 64 - CL : lane < CL) {
            store_floats<V>(lp + w * kChannels + cl * V, P);
            store_floats<V>(lh + w * kChannels + cl * V, H);
        }
        // Of the lanes before this one alone.
        float p0[V], h0[V];
        const bool first = kUp ? lane < CL : lane >= 64 - CL;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float p = kUp ? __shfl_up(P[j], CL & 63) : __shfl_down(P[j], CL & 63);
            const float h = kUp ? __shfl_up(H[j], CL & 63) : __shfl_down(H[j], CL & 63);
            p0[j] = first ? 1.f : p;
            h0[j] = first ? 0.f : h;
        }
        __syncthreads();
        float mine[V];
        // Two waves' pairs in flight (all eight took 64 registers).
#pragma unroll 2
        for (int i = 0; i < kWaves; ++i) {
            const int o = kUp ? i : kWaves - 1 - i;
            float p[V], h[V];
            load_floats<V>(p, lp + o * kChannels + cl * V);
            load_floats<V>(h, lh + o * kChannels + cl * V);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (o == w) mine[j] = carry[j];
                carry[j] = fmaf(p[j], carry[j], h[j]);
                if constexpr (kProduct) product[j] *= p[j];
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) start[j] = fmaf(p0[j], mine[j], h0[j]);
    }
};

// The state a segment starts from: `carry` taken through the pairs of the
// segments before it (kUp: 0 .. seg - 1; else segs - 1 .. seg + 1), each token
// lane joining a run of them.
template <typename S, int V, bool kUp>
__device__ __forceinline__ void through_segments(float (&carry)[V], const float* pairs, int64_t n, int64_t D, int64_t c,
                                                 int seg, int segs, int tl, float* lds) {
    const int count = kUp ? seg : segs - 1 - seg, first = kUp ? 0 : seg + 1;
    const int per = (count + S::kTokenLanes - 1) / S::kTokenLanes;
    float P[V], H[V];
#pragma unroll
    for (int j = 0; j < V; ++j) P[j] = 1.f, H[j] = 0.f;
    for (int i = 0; i < per; ++i) {
        const int at = tl * per + (kUp ? i : per - 1 - i);
        if (at >= count || c >= D) continue;
        const float* r = pairs + ((n * segs + first + at) * 2) * D + c;
        float p[V], h[V];
        load_floats<V>(p, r);
        load_floats<V>(h, r + D);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            H[j] = fmaf(p[j], H[j], h[j]);
            P[j] *= p[j];
        }
    }
    float start[V], none[V];
    S::template join<kUp, false>(P, H, carry, start, none, lds);
}

// One workgroup per (block of channels, stream, segment).  kPairs: only the
// segment's pair, into a.pairs.
template <typename TIn, int V, int CL, int NT, int R, int RB, int kForm, bool kComplement, bool kPairs, int kPolicy>
__global__ __launch_bounds__(NT) void scan_forward_kernel(const ScanGeo g, const ScanFwdArgs a) {
    using S = ScanTile<NT, CL, R, V>;
    using X = Piece<TIn, V>;
    __shared__ __align__(16) float lds[S::kLdsFloats];
    const int cl = threadIdx.x % CL, tl = threadIdx.x / CL;
    const int64_t n = blockIdx.y, D = g.D;
    const int seg = blockIdx.z;
    const int64_t c = (int64_t(blockIdx.x) * CL + cl) * V;
    const bool mine = c < D;
    const int64_t t0 = seg * g.seg_len, t1 = min(g.T, t0 + g.seg_len), end = min(t1, g.live.of(n, g.T));
    const TIn* xp = static_cast<const TIn*>(a.x) + n * g.xn;
    const TIn* gp = static_cast<const TIn*>(a.gate) + n * g.gn;
    TIn* op = static_cast<TIn*>(a.out) + n * g.T * D;
    // Byte offsets of this thread's first row in a tile; a thread past the
    // channels reads zeros and writes nothing.
    constexpr int es = int(sizeof(TIn));
    const int xs = int(g.xt) * es, gs = int(g.gt) * es, os = int(D) * es;
    const int xo = mine ? tl * R * xs + int(c) * es : kPastTile;
    const int go = mine ? tl * R * gs + int(c) * es : kPastTile;
    const int oo = mine ? tl * R * os + int(c) * es : kPastTile;
    X xn[R], gn[R];
    auto load = [&](int64_t r0) {
        const auto xr = rows_view<S::kTile>(xp, r0, end, g.xt, D);
        const auto gr = rows_view<S::kTile>(gp, r0, end, g.gt, D);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            xn[r].template load<kPolicy>(xr, xo + r * xs);
            gn[r].template load<kPolicy>(gr, go + r * gs);
        }
    };
    if (t0 < end) load(t0);
    float carry[V], product[V], start[V];
#pragma unroll
    for (int j = 0; j < V; ++j) carry[j] = 0.f, product[j] = 1.f;
    int parity = 0;
    if constexpr (!kPairs) {
        if (a.state_in && mine) load_floats<V>(carry, a.state_in + n * D + c);
        if (seg > 0) {
            through_segments<S, V, true>(carry, a.pairs, n, D, c, seg, g.segs, tl, lds);
            parity = 1;
        }
    }
    for (int64_t r0 = t0; r0 < t1; r0 += S::kTile) {
        const int64_t t = r0 + tl * R;
        if (r0 >= end) {  // nothing live from here on
            if constexpr (kPairs) break;
            const float zero[V] = {};
            const auto orr = rows_view<S::kTile>(op, r0, t1, D, D);
#pragma unroll
            for (int r = 0; r < R; ++r) X::template store<kPolicy>(orr, oo + r * os, zero);
            continue;
        }
        float av[R][V], uv[R][V], P[V], H[V];
#pragma unroll
        for (int j = 0; j < V; ++j) P[j] = 1.f, H[j] = 0.f;
        const bool whole = r0 + S::kTile <= end;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float b;
                open_gate<kForm>(gn[r].get(j), av[r][j], b);
                uv[r][j] = kComplement ? b * xn[r].get(j) : xn[r].get(j);
            }
        if (!whole) {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    av[r][j] = t + r < end ? av[r][j] : 1.f;
                    uv[r][j] = t + r < end ? uv[r][j] : 0.f;
                }
        }
        if (r0 + S::kTile < end) load(r0 + S::kTile);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                H[j] = fmaf(av[r][j], H[j], uv[r][j]);
                P[j] *= av[r][j];
            }
        S::template join<true, kPairs>(P, H, carry, start, product, lds + parity * (S::kLdsFloats / 2));
        parity ^= 1;
        if constexpr (!kPairs) {
            constexpr int kRecord = S::kTokenLanes * RB;  // tokens of a backward tile
            static_assert(kRecord % R == 0 && S::kTile % kRecord == 0, "a thread's tokens start a record or do not");
            if (a.records && mine && tl * R % kRecord == 0 && t < end)
                store_floats<V>(a.records + (n * g.tiles + t / kRecord) * D + c, start);
            const auto orr = rows_view<S::kTile>(op, r0, t1, D, D);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float y[V];
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    start[j] = fmaf(av[r][j], start[j], uv[r][j]);
                    y[j] = whole || t + r < end ? start[j] : 0.f;
                }
                X::template store<kPolicy>(orr, oo + r * os, y);
            }
        }
    }
    if (!mine || tl != 0) return;
    if constexpr (kPairs) {
        float* r = a.pairs + ((n * g.segs + seg) * 2) * D + c;
        store_floats<V>(r, product);
        store_floats<V>(r + D, carry);
    } else {
        if (a.state_out && seg == g.segs - 1) store_floats<V>(a.state_out + n * D + c, carry);
    }
}

// The gradients, tiles and segments from the last to the first.
template <typename TIn, int V, int CL, int NT, int R, int kForm, bool kComplement, bool kPairs, int kPolicy>
__global__ __launch_bounds__(NT) void scan_backward_kernel(const ScanGeo g, const ScanBwdArgs a) {
    using S = ScanTile<NT, CL, R, V>;
    using X = Piece<TIn, V>;
    __shared__ __align__(16) float lds[S::kLdsFloats];
    const int cl = threadIdx.x % CL, tl = threadIdx.x / CL;
    const int64_t n = blockIdx.y, D = g.D;
    const int seg = blockIdx.z;
    const int64_t c = (int64_t(blockIdx.x) * CL + cl) * V;
    const bool mine = c < D;
    const int64_t t0 = seg * g.seg_len, t1 = min(g.T, t0 + g.seg_len), end = min(t1, g.live.of(n, g.T));
    const TIn* xp = static_cast<const TIn*>(a.x) + n * g.xn;
    const TIn* gp = static_cast<const TIn*>(a.gate) + n * g.gn;
    const TIn* yp = static_cast<const TIn*>(a.dout) + n * g.T * D;
    const float* hp = kPairs ? nullptr : a.records + n * g.tiles * D + c;
    TIn* dxp = a.dx ? static_cast<TIn*>(a.dx) + n * g.T * D : nullptr;
    TIn* dgp = a.dgate ? static_cast<TIn*>(a.dgate) + n * g.T * D : nullptr;
    constexpr int es = int(sizeof(TIn));
    const int xs = int(g.xt) * es, gs = int(g.gt) * es, os = int(D) * es;
    const int xo = mine ? tl * R * xs + int(c) * es : kPastTile;
    const int go = mine ? tl * R * gs + int(c) * es : kPastTile;
    const int oo = mine ? tl * R * os + int(c) * es : kPastTile;
    X xn[R], gn[R], yn[R];
    float hn[V] = {};
    auto load = [&](int64_t r0) {
        if constexpr (!kPairs) {
            if (mine) load_floats<V>(hn, hp + r0 / S::kTile * D);
        }
        const auto xr = rows_view<S::kTile>(xp, r0, end, g.xt, D);
        const auto gr = rows_view<S::kTile>(gp, r0, end, g.gt, D);
        const auto yr = rows_view<S::kTile>(yp, r0, end, D, D);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if constexpr (!kPairs) xn[r].template load<kPolicy>(xr, xo + r * xs);
            gn[r].template load<kPolicy>(gr, go + r * gs);
            yn[r].template load<kPolicy>(yr, oo + r * os);
        }
    };
    // A gradient that is not asked for: a view of no rows.
    auto out_view = [&](TIn* p, int64_t r0) { return rows_view<S::kTile>(p, p ? r0 : 0, p ? t1 : 0, D, D); };
    const int64_t last_tile = t0 + (t1 - 1 - t0) / S::kTile * S::kTile;       // of the segment
    const int64_t last_live = t0 + (end - 1 - t0) / S::kTile * S::kTile;      // where end > t0
    if (t0 < end) load(last_live);
    float carry[V], product[V], start[V];
#pragma unroll
    for (int j = 0; j < V; ++j) carry[j] = 0.f, product[j] = 1.f;
    int parity = 0;
    if constexpr (!kPairs) {
        if (a.dfinal && mine) load_floats<V>(carry, a.dfinal + n * D + c);
        if (seg < g.segs - 1) {
            through_segments<S, V, false>(carry, a.pairs, n, D, c, seg, g.segs, tl, lds);
            parity = 1;
        }
    }
    for (int64_t r0 = last_tile; r0 >= t0; r0 -= S::kTile) {
        const int64_t t = r0 + tl * R;
        if (r0 >= end) {
            if constexpr (kPairs) continue;
            const float zero[V] = {};
            const auto dxr = out_view(dxp, r0), dgr = out_view(dgp, r0);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                X::template store<kPolicy>(dxr, oo + r * os, zero);
                X::template store<kPolicy>(dgr, oo + r * os, zero);
            }
            continue;
        }
        const bool whole = r0 + S::kTile <= end;
        float av[R][V], bv[R][V], ev[R][V], yv[R][V], P[V], H[V];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                open_gate<kForm>(gn[r].get(j), av[r][j], bv[r][j]);
                yv[r][j] = yn[r].get(j);
                if constexpr (!kPairs) ev[r][j] = xn[r].get(j);
            }
        if (!whole) {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const bool live = t + r < end;
                    av[r][j] = live ? av[r][j] : 1.f;
                    bv[r][j] = live ? bv[r][j] : 0.f;
                    yv[r][j] = live ? yv[r][j] : 0.f;
                    if constexpr (!kPairs) ev[r][j] = live ? ev[r][j] : 0.f;
                }
        }
        float h[V];
        if constexpr (!kPairs) {
#pragma unroll
            for (int j = 0; j < V; ++j) h[j] = hn[j];
        }
        if (r0 > t0) load(r0 - S::kTile);
        if constexpr (!kPairs) {
            // h before each token, from the tile's record; then ev = what lambda_t
            // is multiplied with in the gate's gradient.
#pragma unroll
            for (int j = 0; j < V; ++j) P[j] = 1.f, H[j] = 0.f;
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float u = kComplement ? bv[r][j] * ev[r][j] : ev[r][j];
                    H[j] = fmaf(av[r][j], H[j], u);
                    P[j] *= av[r][j];
                }
            float none[V];
            S::template join<true, false>(P, H, h, start, none, lds + parity * (S::kLdsFloats / 2));
            parity ^= 1;
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float x = ev[r][j], before = start[j];
                    start[j] = fmaf(av[r][j], before, kComplement ? bv[r][j] * x : x);
                    const float dlog = av[r][j] * (kComplement ? before - x : before);
                    ev[r][j] = kForm == RACE_GATE_SIGMOID ? bv[r][j] * dlog : dlog;
                }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) P[j] = 1.f, H[j] = 0.f;
#pragma unroll
        for (int r = R - 1; r >= 0; --r)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                H[j] = av[r][j] * (H[j] + yv[r][j]);
                P[j] *= av[r][j];
            }
        S::template join<false, kPairs>(P, H, carry, start, product, lds + parity * (S::kLdsFloats / 2));
        parity ^= 1;
        if constexpr (!kPairs) {
            const auto dxr = out_view(dxp, r0), dgr = out_view(dgp, r0);
#pragma unroll
            for (int r = R - 1; r >= 0; --r) {
                float dx[V], dg[V];
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float lam = start[j] + yv[r][j];
                    start[j] = av[r][j] * lam;
                    dx[j] = kComplement ? bv[r][j] * lam : lam;
                    dg[j] = ev[r][j] * lam;
                }
                if (!whole) {
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        dx[j] = t + r < end ? dx[j] : 0.f;
                        dg[j] = t + r < end ? dg[j] : 0.f;
                    }
                }
                X::template store<kPolicy>(dxr, oo + r * os, dx);
                X::template store<kPolicy>(dgr, oo + r * os, dg);
            }
        }
    }
    if (!mine || tl != 0) return;
    if constexpr (kPairs) {
        float* r = a.pairs + ((n * g.segs + seg) * 2) * D + c;
        store_floats<V>(r, product);
        store_floats<V>(r + D, carry);
    } else {
        if (a.dstate && seg == 0) store_floats<V>(a.dstate + n * D + c, carry);
    }
}

// A few tokens (decode): V channels of a stream per thread, token by token.
// state_out may be state_in.
template <typename TIn, int V, int kForm, bool kComplement>
__global__ __launch_bounds__(kThreads) void scan_step_kernel(const ScanGeo g, const ScanFwdArgs a, int64_t N) {
    using X = Piece<TIn, V>;
    const int64_t per = g.D / V, i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
    if (i >= N * per) return;
    const int64_t n = i / per, c = (i - n * per) * V;
    const int64_t end = g.live.of(n, g.T);
    const TIn* xp = static_cast<const TIn*>(a.x) + n * g.xn + c;
    const TIn* gp = static_cast<const TIn*>(a.gate) + n * g.gn + c;
    TIn* op = static_cast<TIn*>(a.out) + n * g.T * g.D + c;
    float h[V];
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = 0.f;
    if (a.state_in) load_floats<V>(h, a.state_in + n * g.D + c);
    for (int64_t t = 0; t < end; ++t) {
        X x, gate;
        x.v = *reinterpret_cast<const typename X::Raw*>(xp + t * g.xt);
        gate.v = *reinterpret_cast<const typename X::Raw*>(gp + t * g.gt);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float av, b;
            open_gate<kForm>(gate.get(j), av, b);
            h[j] = fmaf(av, h[j], kComplement ? b * x.get(j) : x.get(j));
        }
        X::put(op + t * g.D, h);
    }
    const float zero[V] = {};
    for (int64_t t = end; t < g.T; ++t) X::put(op + t * g.D, zero);
    if (a.state_out) store_floats<V>(a.state_out + n * g.D + c, h);
}

// Workgroup shapes: CL lanes across the channels, NF and NB threads forward
// and backward.  Measured in us, forward / backward:
//   32 x 2048 tokens of 2048 bf16 channels, row pieces of 256 bytes (CL 32)
//     155 / 284 with 512 threads, 166 / 267 with 256; of 128 bytes (CL 16)
//     171 / 323 with 512;
//   8 x 4096 x 2048, 256 workgroups of CL 16 or 128 of CL 32: 98 / 170 (512
//     threads), 113 / 203 (256) and 168 / 207;
//   8 x 65536 x 64 (segments): 84 / 120 with 512 threads, 79 / 110 with 256;
//   2 x 4096 x 2048 (segments): CL 32 46 / 60 and 41 / 53, CL 16 49 / 65.
// Per thread 8 tokens forward and 4 backward, which holds four values an
// element: with 8 it spilled 640 bytes a lane (8 x 4096 x 2048: 746 us).
template <int V_, int CL, int NF, int NB, int RF = 8, int RB = 4>
struct ScanShape {
    static constexpr int V = V_, kLanes = CL, kFwdThreads = NF, kBwdThreads = NB, kFwdRun = RF, kBwdRun = RB;
    using Fwd = ScanTile<NF, CL, RF, V>;
    using Bwd = ScanTile<NB, CL, RB, V>;
    static constexpr int kChannels = CL * V;
};
using Wide = ScanShape<4, 32, 512, 256>;
using WideSplit = ScanShape<4, 32, 256, 256>;
using Narrow = ScanShape<4, 16, 512, 512>;
using NarrowSplit = ScanShape<4, 16, 256, 256>;
using Single = ScanShape<1, 64, 512, 512, 8, 8>;  // any strides and widths

// Workgroups from which the tokens are not split, those of 128 channels that are
// taken before those of 64, and those a split aims for; two tiles are never split.
// Whole and split in us, forward and with the backward, by the workgroups of 64
// channels (8 x 4096 tokens in bf16, then 8 x 4096 and 24 x 1531 in fp32):
//   128    77 / 223 and 74 / 172     98 / 276 and 113 / 260
//   144    75 / 222 and 88 / 205     96 / 273 and 126 / 300     39 / 106 and 51 / 118
//   160    78 / 225 and 96 / 222    108 / 310 and 147 / 357
//   168    75 / 222 and 105 / 257                               40 / 110 and 65 / 142
//   192    80 / 238 and 102 / 260   121 / 328 and 164 / 407     48 / 123 and 75 / 159
// from 168 on every call gains (at 160, 2 x 32768 tokens in bf16 trained in 1930
// whole and 1750 split).  Of 128 channels 104 workgroups took 133 / 486 where 200 of
// 64 took 75 / 225.  A split costs a launch, two tiles cost less (10 x 160 x 24, two
// tiles, 7.6 + 11.2 whole and 9.9 + 13.3 split; 2 x 290 x 64, three, 10.2 + 17.3 and
// 9.5 + 13.0).
constexpr int64_t kScanEnough = 168, kScanWide = 200, kScanSplit = 512, kScanWhole = 2;

int64_t blocks_of(const GatedScan& s, int64_t channels) { return s.N * ((s.D + channels - 1) / channels); }

bool scan_vectors(const GatedScan& s) {
    return s.D % 4 == 0 && s.xn % 4 == 0 && s.xt % 4 == 0 && s.gn % 4 == 0 && s.gt % 4 == 0;
}

// f(shape) for the shape of these arguments.
template <typename F>
auto by_shape(const GatedScan& s, F f) {
    if (!scan_vectors(s)) return f(Single{});
    if (blocks_of(s, Wide::kChannels) >= kScanWide) return f(Wide{});
    if (blocks_of(s, Narrow::kChannels) >= kScanEnough) return f(Narrow{});
    return s.D > 96 ? f(WideSplit{}) : f(NarrowSplit{});
}

// Tokens a segment is made of.
int64_t forward_tile(const GatedScan& s) {
    return by_shape(s, [](auto shape) { return int64_t(decltype(shape)::Fwd::kTile); });
}

ScanGeo geometry(const GatedScan& s) {
    ScanGeo g;
    g.T = s.T;
    g.D = s.D;
    g.xn = s.xn, g.xt = s.xt, g.gn = s.gn, g.gt = s.gt;
    g.live = s.live;
    g.tiles = scan_tiles(s);
    g.segs = int(scan_segments(s));
    const int64_t tile = forward_tile(s);
    g.seg_len = ((s.T + tile - 1) / tile + g.segs - 1) / g.segs * tile;
    return g;
}

// f(form, complement) as compile-time values.
template <typename F>
hipError_t by_gate(const GatedScan& s, F f) {
    using Sig = std::integral_constant<int, RACE_GATE_SIGMOID>;
    using Log = std::integral_constant<int, RACE_GATE_LOG>;
    if (s.form == RACE_GATE_SIGMOID) return s.complement ? f(Sig{}, std::true_type{}) : f(Sig{}, std::false_type{});
    return s.complement ? f(Log{}, std::true_type{}) : f(Log{}, std::false_type{});
}

// Calls whose `arrays` row arrays are larger than the memory-side cache holds
// go past the caches, if their rows are whole cache lines: 8 x 4096 x 2048 bf16,
// forward / backward, 105 / 181 us through them and 98 / 170 past them; 1 x
// 32768 x 1024 fp32 139 / 182 and 122 / 158; but 24 x 1531 x 520 fp32, whose
// workgroups share lines, 55 / 99 and 68 / 119.
bool past_scan_caches(const GatedScan& s, int arrays) {
    constexpr int64_t kCacheBytes = int64_t(256) << 20, kLine = 128;
    const int64_t row = s.D * (s.dtype == RACE_BF16 ? 2 : 4);
    return row % kLine == 0 && s.N * s.T * row * arrays > kCacheBytes;
}

template <typename TIn, typename Sh>
hipError_t launch_forward(const GatedScan& s, const ScanFwdArgs& a, hipStream_t stream) {
    constexpr int V = Sh::V, CL = Sh::kLanes, NT = Sh::kFwdThreads, R = Sh::kFwdRun, RB = Sh::Bwd::kTile * CL / NT;
    const ScanGeo g = geometry(s);
    const dim3 grid(unsigned((s.D + Sh::kChannels - 1) / Sh::kChannels), unsigned(s.N), unsigned(g.segs));
    return by_gate(s, [&](auto form, auto comp) {
        // The pairs' reads stay in the caches for the pass that reads the rows again.
        if (g.segs > 1) {
            scan_forward_kernel<TIn, V, CL, NT, R, RB, form.value, comp.value, true, mfma::kPolicyDefault>
                <<<grid, NT, 0, stream>>>(g, a);
            const hipError_t err = hipGetLastError();
            if (err != hipSuccess) return err;
        }
        if (past_scan_caches(s, 3))
            scan_forward_kernel<TIn, V, CL, NT, R, RB, form.value, comp.value, false, mfma::kPolicyStream>
                <<<grid, NT, 0, stream>>>(g, a);
        else
            scan_forward_kernel<TIn, V, CL, NT, R, RB, form.value, comp.value, false, mfma::kPolicyDefault>
                <<<grid, NT, 0, stream>>>(g, a);
        return hipGetLastError();
    });
}

template <typename TIn, typename Sh>
hipError_t launch_backward(const GatedScan& s, const ScanBwdArgs& a, hipStream_t stream) {
    constexpr int V = Sh::V, CL = Sh::kLanes, NT = Sh::kBwdThreads, R = Sh::kBwdRun;
    const ScanGeo g = geometry(s);
    const dim3 grid(unsigned((s.D + Sh::kChannels - 1) / Sh::kChannels), unsigned(s.N), unsigned(g.segs));
    return by_gate(s, [&](auto form, auto comp) {
        if (g.segs > 1) {
            scan_backward_kernel<TIn, V, CL, NT, R, form.value, comp.value, true, mfma::kPolicyDefault>
                <<<grid, NT, 0, stream>>>(g, a);
            const hipError_t err = hipGetLastError();
            if (err != hipSuccess) return err;
        }
        if (past_scan_caches(s, 5))
            scan_backward_kernel<TIn, V, CL, NT, R, form.value, comp.value, false, mfma::kPolicyStream>
                <<<grid, NT, 0, stream>>>(g, a);
        else
            scan_backward_kernel<TIn, V, CL, NT, R, form.value, comp.value, false, mfma::kPolicyDefault>
                <<<grid, NT, 0, stream>>>(g, a);
        return hipGetLastError();
    });
}

template <typename TIn, int V>
hipError_t launch_step_v(const GatedScan& s, const ScanFwdArgs& a, hipStream_t stream) {
    const ScanGeo g = geometry(s);
    const int64_t threads = s.N * (s.D / V);
    return by_gate(s, [&](auto form, auto comp) {
        scan_step_kernel<TIn, V, form.value, comp.value>
            <<<unsigned((threads + kThreads - 1) / kThreads), kThreads, 0, stream>>>(g, a, s.N);
        return hipGetLastError();
    });
}

}  // namespace

int64_t scan_tile_tokens(const GatedScan& s) {
    return by_shape(s, [](auto shape) { return int64_t(decltype(shape)::Bwd::kTile); });
}

int64_t scan_tiles(const GatedScan& s) {
    const int64_t tile = scan_tile_tokens(s);
    return (s.T + tile - 1) / tile;
}

int64_t scan_segments(const GatedScan& s) {
    const int64_t tile = forward_tile(s), tiles = (s.T + tile - 1) / tile;
    const int64_t base = by_shape(s, [&](auto shape) { return blocks_of(s, decltype(shape)::kChannels); });
    if (base >= kScanEnough || tiles <= kScanWhole) return 1;
    const int64_t per = (tiles + kScanSplit / base - 1) / (kScanSplit / base);  // tiles of a segment
    return (tiles + per - 1) / per;
}

hipError_t launch_gated_scan(const GatedScan& s, const void* x, const void* gate, const float* state_in, void* out,
                             float* state_out, float* records, float* pairs, hipStream_t stream) {
    const ScanFwdArgs a{x, gate, state_in, out, state_out, records, pairs};
    if (!records && s.T <= kScanStepTokens) {
        const bool four = scan_vectors(s);
        if (s.dtype == RACE_BF16)
            return four ? launch_step_v<bf16_t, 4>(s, a, stream) : launch_step_v<bf16_t, 1>(s, a, stream);
        return four ? launch_step_v<float, 4>(s, a, stream) : launch_step_v<float, 1>(s, a, stream);
    }
    return by_shape(s, [&](auto shape) {
        return s.dtype == RACE_BF16 ? launch_forward<bf16_t, decltype(shape)>(s, a, stream)
                                    : launch_forward<float, decltype(shape)>(s, a, stream);
    });
}

hipError_t launch_gated_scan_bwd(const GatedScan& s, const void* x, const void* gate, const void* dout,
                                 const float* records, const float* dfinal, void* dx, void* dgate, float* dstate,
                                 float* pairs, hipStream_t stream) {
    const ScanBwdArgs a{x, gate, dout, records, dfinal, dx, dgate, dstate, pairs};
    return by_shape(s, [&](auto shape) {
        return s.dtype == RACE_BF16 ? launch_backward<bf16_t, decltype(shape)>(s, a, stream)
                                    : launch_backward<float, decltype(shape)>(s, a, stream);
    });
}

}  // namespace race
