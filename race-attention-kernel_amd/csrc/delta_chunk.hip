// delta_chunk.hip -- the gated delta rule, forward: per stream a state S [dk][dv],
//
//     S_t = a_t S_{t-1} + b_t k_t (v_t - a_t S_{t-1}^T k_t)^T,   o_t = scale S_t^T q_t.
//
// In chunks of 64 tokens, from the state S before the chunk: with G_i the sum of
// log a up to token i, E_i = e^{G_i}, Z_i = e^{G_last - G_i}, Gam_ij = e^{G_i - G_j},
//
//     N_ij = Gam_ij (k_i . k_j) b_j  (j < i),   T = (I + N)^-1,
//     D = V - E K S,   Y = T D                      (the error each token writes),
//     O = scale (E Q S + (Gam o Q K^T) b Y)         (j <= i),
//     S <- e^{G_last} S + K^T (Z b Y).
//
// Two launches.  delta_solve_kernel, a workgroup per chunk, forms T and the
// masked Gam o Q K^T b; all chunks at once.  delta_chunk_kernel walks a stream's
// chunks in order, 16 columns of the state in a wave's registers: the columns of
// S, D, Y and O do not mix, so its waves share the K, Q and T tiles in LDS and
// nothing else, and every product takes its right operand from the accumulators
// before it (delta_tiles.h).
// Precision.  Sums are fp32, and so are the factors of a product that are computed: with
// fp32 rows in fp32 products, with bf16 rows in three parts of bf16 (delta_tiles.h), so
// that a call of bf16 rows gives what one of the same rows in fp32 does, its outputs
// rounded once.  Errors are relative to the terms of a sum: where a chunk overwrites
// what a state held, a rounding of that, 2^-24, is left until the next chunk.  The
// output's own products, whose result is rounded to bf16 right away, take S, Y and M
// in two parts.  Log decays are summed in 64 bits: differences of long sums lose the
// digits the products keep.
// A few tokens (decode) go token by token in 32 bits: delta_step_kernel, bound by the
// states' bytes (1024 streams, 128 x 128: 134 MB, 23 us).
// The walk is bound by its chain of products: a chunk's K S, T D, K^T Z follow one
// another, 4 us with a wave a SIMD, its matrix cores busy for less than a third of it; so
// its waves hold no more than they need, loads for the next chunk go out between the
// stages, and few streams are walked in segments (delta_segment_chunks).  128 streams
// of 4096 bf16 tokens, 128 x 128, with records: solve 113 us, walk 411 us.
#include <algorithm>
#include <utility>

#include "delta_tiles.h"

namespace race {
namespace {

using namespace delta;
using mfma::mfma4;

// ---- T and the masked scores of a chunk ----

constexpr int kSolvePitch = 68;
constexpr int kSolveMatrix = kChunk * kSolvePitch * 4;

template <typename TIn, int DK>
constexpr int solve_lds_bytes() {
    constexpr int tiles = 2 * Tile<TIn, DK>::kBytes;
    return tiles > 2 * kSolveMatrix ? tiles : 2 * kSolveMatrix;
}

// acc += X[r0 ..][c0 ..] B for 16 x 16 fp32 blocks, B in accumulator order.
__device__ __forceinline__ f32x4 block_times(const float* x, int r0, int c0, int g, int lr, const f32x4& b, f32x4 acc) {
    const float4 a = *reinterpret_cast<const float4*>(x + (r0 + lr) * kSolvePitch + c0 + 4 * g);
    acc = mfma4(a.x, b[0], acc);
    acc = mfma4(a.y, b[1], acc);
    acc = mfma4(a.z, b[2], acc);
    return mfma4(a.w, b[3], acc);
}
__device__ __forceinline__ f32x4 block_of(const float* x, int r0, int c0, int g, int lr) {
    f32x4 v;
#pragma unroll
    for (int s = 0; s < 4; ++s) v[s] = x[(r0 + 4 * g + s) * kSolvePitch + c0 + lr];
    return v;
}

// x -= n_j x_j for every row below j, whose N is zero up to its diagonal: x_j from
// lane j of the lane's 16.
template <int... J>
__device__ __forceinline__ void substitute(f32x4& x, const f32x4 (&n)[4], std::integer_sequence<int, J...>) {
    auto step = [&](auto j) {
        constexpr int kBroadcast = 0x150 + decltype(j)::value;  // row_newbcast
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int v = __float_as_int(x[c]);
            x[c] = fmaf(-n[decltype(j)::value / 4][decltype(j)::value % 4],
                        __int_as_float(__builtin_amdgcn_update_dpp(v, v, kBroadcast, 0xf, 0xf, true)), x[c]);
        }
    };
    (step(std::integral_constant<int, J>{}), ...);
}

template <typename TIn, int DK, bool kVec>
__global__ __launch_bounds__(kThreads, sizeof(TIn) * DK <= 256 ? 4 : 2) void delta_solve_kernel(const DeltaArgs a) {
    extern __shared__ __align__(16) unsigned char lds[];
    __shared__ __align__(16) double G[kChunk];
    __shared__ __align__(16) float b[kChunk];
    using Rows = Tile<TIn, DK>;
    unsigned char *kt = lds, *qt = lds + Rows::kBytes;
    // Over the tiles, once they are read.
    float *T = reinterpret_cast<float*>(lds), *Nm = reinterpret_cast<float*>(lds + kSolveMatrix);
    const int64_t nc = blockIdx.x, n = blockIdx.x / unsigned(a.chunks);
    const int t0 = int(nc - n * a.chunks) * kChunk;
    const int64_t len = a.len_of(n);
    if (t0 >= len) return;
    const int live = int(len - t0 < kChunk ? len - t0 : kChunk);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, lr = lane & 15;
    const int64_t nk = a.key_stream(n);
    auto row_of = [&](const unsigned char* t, int row, int s) { return Rows::load(t, Rows::run_at(row, 4 * s + g)); };
    {
        Stage<TIn, DK, kThreads, kVec> k, q;
        k.init(a.kt, a.dk);
        q.init(a.qt, a.dk);
        const int64_t at = n * a.T + t0 + min(lane, live - 1);
        const uint32_t gate = a.gate ? gate_bits(a.gate, at, a.gate_f32) : 0, beta = gate_bits(a.beta, at, a.gate_f32);
        k.load(static_cast<const TIn*>(a.k) + nk * a.kn + t0 * a.kt, live);
        q.load(static_cast<const TIn*>(a.q) + nk * a.qn + t0 * a.qt, live);
        if (wave == 0) {
            double s = double(log_decay(gate_of(gate, a.gate_f32), a.form)) * kLog2e;
            s = wave_scan(lane < live && a.gate ? s : 0.0);
            G[lane] = s;
            const float bv = lane < live ? gate_of(beta, a.gate_f32) : 0.f;
            b[lane] = bv;
            const double last = __shfl(s, 63);
            float* vec = a.vec + nc * 128;
            vec[lane] = __builtin_amdgcn_exp2f(float(s));
            vec[64 + lane] = __builtin_amdgcn_exp2f(float(last - s)) * bv;
        }
        k.put(kt);
        q.put(qt);
    }
    __syncthreads();
    // Row block `wave` of K K^T, `o` of Q K^T, a token's columns in a lane.  bf16 products of the blocks above the diagonal
    // cost less than branches around them; fp32 ones are left out, five blocks a wave in all.
    constexpr bool kAll = sizeof(TIn) == 2;
    const int o = kAll ? wave : 3 - wave;
    f32x4 kk[4], qk[4];
    {
        decltype(row_of(kt, 0, 0)) kr[DK / 32], qr[DK / 32];
#pragma unroll
        for (int s = 0; s < DK / 32; ++s) kr[s] = row_of(kt, 16 * wave + lr, s), qr[s] = row_of(qt, 16 * o + lr, s);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            kk[j] = qk[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < DK / 32; ++s) {
                const auto kj = row_of(kt, 16 * j + lr, s);
                if (kAll || j <= wave) kk[j] = mac(kj, kr[s], kk[j]);
                if (kAll || j <= o) qk[j] = mac(kj, qr[s], qk[j]);
            }
        }
    }
    // Gam b of a row of block `block` and four columns: kept for N where both are of the same rows.
    auto weights = [&](int block, int j) {
        const int col = 16 * j + 4 * g;
        const double gr = G[16 * block + lr];
        const double2 g0 = *reinterpret_cast<const double2*>(G + col), g1 = *reinterpret_cast<const double2*>(G + col + 2);
        const f32x4 e = {float(gr - g0.x), float(gr - g0.y), float(gr - g1.x), float(gr - g1.y)};
        f32x4 x = *reinterpret_cast<const f32x4*>(b + col);
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] *= __builtin_amdgcn_exp2f(e[r]);
        return x;
    };
    auto below = [&](int block, int j, f32x4 x, int first) {  // zero past the row's token, or from it on
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = 16 * block + lr >= 16 * j + 4 * g + r + first ? x[r] : 0.f;
        return x;
    };
    f32x4 gb[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        gb[j] = weights(o, j);
        if (j <= (o | 1))  // the others are not read
            SquareOf<TIn>::put4(a.mm + nc * SquareOf<TIn>::kBytes, 16 * o + lr, 16 * j + 4 * g, below(o, j, gb[j] * qk[j] * a.scale, 0),
                                a.st ? 3 : 2);  // the third part is the backward's
        if (!kAll) gb[j] = weights(wave, j);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j)
        *reinterpret_cast<f32x4*>(Nm + (16 * wave + lr) * kSolvePitch + 16 * j + 4 * g) = below(wave, j, gb[j] * kk[j], 1);
    __syncthreads();
    // (I + N)^-1: the diagonal blocks by substitution, rows in the lanes of a row of
    // 16 and four columns in each, ...
    {
        const int r0 = 16 * wave;
        f32x4 n[4], x;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            n[j] = *reinterpret_cast<const f32x4*>(Nm + (r0 + lr) * kSolvePitch + r0 + 4 * j);
#pragma unroll
        for (int c = 0; c < 4; ++c) x[c] = lr == 4 * g + c ? 1.f : 0.f;
        substitute(x, n, std::make_integer_sequence<int, 15>{});
        *reinterpret_cast<f32x4*>(T + (r0 + lr) * kSolvePitch + r0 + 4 * g) = x;
    }
    __syncthreads();
    // ... then [A 0; C B]^-1 = [A' 0; -B' C A'  B'], of 16 and of 32 rows.
    if (wave < 2) {
        const int r0 = 32 * wave;
        f32x4 w = {0.f, 0.f, 0.f, 0.f}, z = w;
        w = block_times(Nm, r0 + 16, r0, g, lr, block_of(T, r0, r0, g, lr), w);
        z = block_times(T, r0 + 16, r0 + 16, g, lr, w, z);
#pragma unroll
        for (int r = 0; r < 4; ++r) T[(r0 + 16 + 4 * g + r) * kSolvePitch + r0 + lr] = -z[r];
    }
    __syncthreads();
    {
        const int i = wave >> 1, j = wave & 1;
        f32x4 z = {0.f, 0.f, 0.f, 0.f};
        f32x4 from[2];
#pragma unroll
        for (int l = 0; l < 2; ++l)
            if (l >= j) from[l] = block_of(T, 16 * l, 16 * j, g, lr);
        for (int k = 0; k <= i; ++k) {
            f32x4 w = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int l = 0; l < 2; ++l)
                if (l >= j) w = block_times(Nm, 32 + 16 * k, 16 * l, g, lr, from[l], w);
            z = block_times(T, 32 + 16 * i, 32 + 16 * k, g, lr, w, z);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) T[(32 + 16 * i + 4 * g + r) * kSolvePitch + 16 * j + lr] = -z[r];
    }
    __syncthreads();
    const int row = threadIdx.x >> 2, c0 = (threadIdx.x & 3) * 16;
    unsigned char* tm = a.tm + nc * SquareOf<TIn>::kBytes;
#pragma unroll
    for (int e = 0; e < 16; e += 8) {
        f32x4 x[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            x[h] = *reinterpret_cast<const f32x4*>(T + row * kSolvePitch + c0 + e + 4 * h);
#pragma unroll
            for (int r = 0; r < 4; ++r) x[h][r] = c0 + e + 4 * h + r <= row ? x[h][r] : 0.f;
        }
        SquareOf<TIn>::put8(tm, row, c0 + e, x[0], x[1]);
    }
}

// ---- the walk over a stream's chunks ----

// What a walk leaves: outputs; outputs and the records of a backward; or, in place
// of outputs, what its segment does to a state: columns of the identity (with
// values of zero) beside those of the values (from zero, the first segment's from
// its state).
enum WalkMode { kOutputs, kRecording, kMaps };

template <typename TIn, int DK, WalkMode kMode>
using WalkLds = ChunkLds<TIn, DK, 2, kMode != kMaps, !two_a_cu(sizeof(TIn) * DK, kMode == kMaps)>;

// kVec, kVecV: rows of keys, and of values and outputs, in 16-byte pieces.
template <typename TIn, int DK, bool kVec, bool kVecV, WalkMode kMode>
__global__ __launch_bounds__(kThreads, two_a_cu(sizeof(TIn) * DK, kMode == kMaps) ? 2 : 1) void delta_chunk_kernel(const DeltaArgs a) {
    extern __shared__ __align__(16) unsigned char lds[];
    using L = WalkLds<TIn, DK, kMode>;
    constexpr bool kLate = two_a_cu(sizeof(TIn) * DK, kMode == kMaps) && kMode != kMaps;
    using Rows = Tile<TIn, DK>;
    using Square = Tile<TIn, 64>;
    using One = OneT<TIn>;
    using Two = TwoT<TIn>;
    using Three = ThreeT<TIn>;
    constexpr int NS = DK / 32;
    const int value_blocks = (a.dv + 63) / 64, blocks = value_blocks + (kMode == kMaps ? (a.dk + 63) / 64 : 0);
    const int walks = kMode == kMaps ? a.segs - 1 : a.segs;  // no state follows the last segment's
    int64_t ns;
    int cb;
    if (!stream_and_block(a.N * walks, blocks, ns, cb)) return;
    const int64_t n = unsigned(ns) / unsigned(walks);
    const int seg = int(ns - n * walks);
    const bool unit = kMode == kMaps && cb >= value_blocks;
    if (unit && seg == 0) return;  // its start is known
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, lr = lane & 15;
    const bool odd = g & 1;
    const int width = unit ? a.dk : a.dv, values = unit ? 0 : a.dv - cb * 64;
    const int c0 = (unit ? cb - value_blocks : cb) * 64 + wave * 16, col = c0 + lr;
    const bool active = c0 < width;
    const int64_t nk = a.key_stream(n), len = a.len_of(n);
    const int all = int((len + kChunk - 1) / kChunk);
    const int from = min(seg * a.seg_chunks, all), chunks = min(from + a.seg_chunks, all);
    const TIn* kp = static_cast<const TIn*>(a.k) + nk * a.kn;
    const TIn* qp = static_cast<const TIn*>(a.q) + nk * a.qn;
    const TIn* vp = static_cast<const TIn*>(a.v) + n * a.vn + (unit ? 0 : cb * 64);
    TIn* op = static_cast<TIn*>(a.out) + n * a.T * a.dv;
    const float* start = kMode != kMaps && a.starts ? a.starts + ns * a.dk * a.dv
                         : a.state && seg == 0      ? a.state + n * a.dk * a.dv
                                                    : nullptr;

    f32x4 S[DK / 16];
    if (start && !unit) {
        const StateView from(start, a.dk, a.dv);
#pragma unroll
        for (int i = 0; i < DK / 16; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) S[i][r] = from.one(tok(i, 4 * g + r), col);
    } else {
#pragma unroll
        for (int i = 0; i < DK / 16; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) S[i][r] = unit && tok(i, 4 * g + r) == col ? 1.f : 0.f;
    }

    Stage<TIn, DK, kThreads, kVec> sk, sq;
    StageSquare<TIn, 3> stm;
    StageSquare<TIn, 2> smm;
    Stage<TIn, 64, kThreads, kVecV> sv;
    float svec;
    sk.init(a.kt, a.dk);
    sq.init(a.qt, a.dk);
    sv.init(a.vt, values);
    // A chunk's loads, in four parts: all at once they fill the queue, and the wave waits to issue them.
    auto fetch = [&](int c, int part) {
        const int64_t nc = n * a.chunks + c, t0 = int64_t(c) * kChunk;
        const int live = int(len - t0 < kChunk ? len - t0 : kChunk);
        if (part == 0) sk.load(kp + t0 * a.kt, live);
        if (part == 1 && kMode != kMaps) sq.load(qp + t0 * a.qt, live);
        if (part == 2) stm.load(a.tm + nc * SquareOf<TIn>::kBytes);
        if (part == 3) {
            if (kMode != kMaps) smm.load(a.mm + nc * SquareOf<TIn>::kBytes);
            sv.load(vp + t0 * a.vt, live);
            svec = a.vec[nc * 128 + (threadIdx.x & 127)];
        }
    };
    // What a lane adds to a tile's start.
    const int k_row = Rows::row_base(lr, g), k_col = Rows::column_base(lr, g), s_row = Square::row_base(lr, g);
    const int v_at = Square::block_base(16 * wave, lr, g);
    if (from < chunks)
        for (int p = 0; p < 4; ++p) fetch(from, p);
    for (int c = from; c < chunks; ++c) {
        unsigned char* buf = lds + (L::kBuffers == 2 ? (c & 1) * L::kBytes : 0);
        if (L::kBuffers == 1 && c > from) __syncthreads();  // the chunk before is done with the buffer
        sk.put(buf + L::kK);
        if (kMode != kMaps) sq.put(buf + L::kQ);
        stm.put(buf + L::kT);
        if (kMode != kMaps) smm.put(buf + L::kM);
        sv.put(buf + L::kV);
        reinterpret_cast<float*>(buf + L::kVec)[threadIdx.x & 127] = svec;
        const int next = c + 1 < chunks ? c + 1 : c;  // the last chunk's loads are not used
        __syncthreads();
        if (!active) {
            for (int p = 0; p < 4; ++p) fetch(next, p);
            continue;
        }
        const float* E = reinterpret_cast<const float*>(buf + L::kVec);
        const int64_t nc = n * a.chunks + c;
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
        One kf[NS][4];
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int b = 0; b < 4; ++b) kf[i][b] = Rows::one(buf + L::kK, k_row, b, i);
        Three s[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) operand(S[2 * i], S[2 * i + 1], odd, s[i]);
        if constexpr (kMode == kRecording) {
            float* st = a.st + (nc * a.dvp + col) * DK + 8 * g;
#pragma unroll
            for (int i = 0; i < NS; ++i) store_run(st + 32 * i, S[2 * i], S[2 * i + 1], odd, s[i]);
        }
        stage_wall();
        fetch(next, 0);
        Three tf[4], tg[2];
        f32x4 e[4], v[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            e[b] = *reinterpret_cast<const f32x4*>(E + tok(b, 4 * g));
            v[b] = Square::block(buf + L::kV, v_at, b);
            tf[b] = Square::template parts<3>(buf + L::kT, s_row, b, 0);
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) tg[b] = Square::template parts<3>(buf + L::kT, s_row, 2 + b, 1);
        // D = V - E K S.
        f32x4 x[4];
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int b = 0; b < 4; ++b) x[b] = mac(kf[i][b], s[i], i == 0 ? zero : x[b]);
        stage_wall();
        fetch(next, 1);
        One kc[2][DK / 16];
        auto columns = [&] {
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int i = 0; i < DK / 16; ++i) kc[kk][i] = Rows::transposed(buf + L::kK, k_col, kk, i);
        };
        if (!kLate) columns();
        f32x4 zb[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) zb[b] = *reinterpret_cast<const f32x4*>(E + 64 + tok(b, 4 * g));
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) x[b][r] = fmaf(-e[b][r], x[b][r], v[b][r]);
        Three d[2];
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) operand(x[2 * kk], x[2 * kk + 1], odd, d[kk]);
        // Y = T D; T is lower triangular.
#pragma unroll
        for (int b = 0; b < 4; ++b) x[b] = mac(tf[b], d[0], zero);
#pragma unroll
        for (int b = 2; b < 4; ++b) x[b] = mac(tg[b - 2], d[1], x[b]);
        stage_wall();
        fetch(next, 2);
        if (kLate) columns();
        One qf[NS][4];
        if constexpr (kMode != kMaps && !kLate) {
#pragma unroll
            for (int i = 0; i < NS; ++i)
#pragma unroll
                for (int b = 0; b < 4; ++b) qf[i][b] = Rows::one(buf + L::kQ, k_row, b, i);
        }
        Two y[2];  // for the output
        Three z[2];
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            operand(x[2 * kk], x[2 * kk + 1], odd, y[kk]);
            operand(x[2 * kk] * zb[2 * kk], x[2 * kk + 1] * zb[2 * kk + 1], odd, z[kk]);
        }
        if constexpr (kMode == kRecording) {
            float* yt = a.yt + (nc * a.dvp + col) * kChunk + 8 * g;
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) store_run(yt + 32 * kk, x[2 * kk], x[2 * kk + 1], odd, y[kk]);
        }
        // S = e^{G_last} S + K^T (Z b Y).
        const float decay = E[63];
#pragma unroll
        for (int i = 0; i < DK / 16; ++i) S[i] *= decay;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
            for (int i = 0; i < DK / 16; ++i) S[i] = mac(kc[kk][i], z[kk], S[i]);
        stage_wall();
        fetch(next, 3);
        if constexpr (kMode == kMaps) continue;
        Two mf[4], mg[2];
        float es[4];
        auto scores = [&] {
#pragma unroll
            for (int b = 0; b < 4; ++b) mf[b] = Square::template parts<2>(buf + L::kM, s_row, b, 0), es[b] = E[tok(b, lr)] * a.scale;
#pragma unroll
            for (int b = 0; b < 2; ++b) mg[b] = Square::template parts<2>(buf + L::kM, s_row, 2 + b, 1);
        };
        if (!kLate) scores();
        // O^T = scale S^T Q^T E + Y^T M^T, S the state before the chunk: a token's columns in a lane.
        f32x4 o[4];
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            if constexpr (kLate) {
#pragma unroll
                for (int b = 0; b < 4; ++b) qf[i][b] = Rows::one(buf + L::kQ, k_row, b, i);
            }
#pragma unroll
            for (int b = 0; b < 4; ++b) o[b] = mac(delta::first<2>(s[i]), qf[i][b], i == 0 ? zero : o[b]);
        }
        if (kLate) scores();
#pragma unroll
        for (int b = 0; b < 4; ++b) o[b] = mac(y[0], mf[b], o[b] * es[b]);
#pragma unroll
        for (int b = 2; b < 4; ++b) o[b] = mac(y[1], mg[b - 2], o[b]);
        const int64_t t0 = int64_t(c) * kChunk;
        // Rows past the last live one lie outside the view.
        const int rows = int(len - t0 < kChunk ? len - t0 : kChunk), bytes = int(sizeof(TIn));
        const auto out = mfma::make_rsrc(op + t0 * a.dv, int64_t(rows) * a.dv * bytes);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int at = (tok(b, lr) * a.dv + c0 + 4 * g) * bytes, there = a.dv - c0 - 4 * g;
            if constexpr (kVecV) {
                mfma::store4<TIn, mfma::kPolicyDefault>(out, there > 0 ? at : mfma::kOutside, o[b]);
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int off = r < there ? at + r * bytes : mfma::kOutside;
                    if constexpr (sizeof(TIn) == 4)
                        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(o[b][r]), out, off, 0, 0);
                    else
                        __builtin_amdgcn_raw_buffer_store_b16(f32_to_bf16(o[b][r]), out, off, 0, 0);
                }
            }
        }
    }
    if (!active || col >= width) return;
    float* to = nullptr;
    if constexpr (kMode == kMaps) {
        const int64_t at = n * a.segs + seg;
        to = unit ? a.map_a + at * a.dk * a.dk : a.map_x + at * a.dk * a.dv;
    } else {
        // The segment's tokens past the stream's last live one.
        const int64_t left = int64_t(seg) * a.seg_chunks * kChunk, right = left + int64_t(a.seg_chunks) * kChunk;
        const int64_t stop = right < a.T ? right : a.T;
        for (int64_t t = (len > left ? len : left) + g; t < stop; t += 4) store_val(op + t * a.dv + col, 0.f);
        const bool last = all == 0 ? seg == 0 : from < all && chunks == all;
        if (last && a.final_state) to = a.final_state + n * a.dk * a.dv;
    }
    if (!to) return;
#pragma unroll
    for (int i = 0; i < DK / 16; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = tok(i, 4 * g + r);
            if (row < a.dk) to[row * width + col] = S[i][r];
        }
}

// ---- token by token ----

// V columns a thread and R rows, every eighth: a workgroup holds 32 V columns of a
// stream's state, all rows.  final_state may be state.
template <typename TIn, int V, int R>
__global__ __launch_bounds__(kThreads) void delta_step_kernel(const DeltaArgs a) {
    constexpr int CQ = 32, RG = kThreads / CQ;
    __shared__ float ks[R * RG], qs[R * RG], sums[4][CQ][2 * V + 1];
    const int64_t n = blockIdx.y, nk = a.key_stream(n), len = a.len_of(n);
    const int cl = threadIdx.x % CQ, rg = threadIdx.x / CQ, wave = threadIdx.x >> 6;
    const int c = (blockIdx.x * CQ + cl) * V;
    const bool in = c < a.dv;
    float S[R][V];
    if (a.state) {
        const StateView from(a.state + n * a.dk * a.dv, a.dk, a.dv);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int row = i * RG + rg;
            if constexpr (V == 4) {
                const f32x4 s = from.four(row, c);
#pragma unroll
                for (int j = 0; j < 4; ++j) S[i][j] = s[j];
            } else {
                S[i][0] = from.one(row, c);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) S[i][j] = 0.f;
    }
    TIn* op = static_cast<TIn*>(a.out) + n * a.T * a.dv + c;
#pragma unroll 1
    for (int64_t t = 0; t < len; ++t) {
        for (int i = threadIdx.x; i < 2 * R * RG; i += kThreads) {
            const bool key = i < R * RG;
            const int row = key ? i : i - R * RG;
            const TIn* p = key ? static_cast<const TIn*>(a.k) + nk * a.kn + t * a.kt : static_cast<const TIn*>(a.q) + nk * a.qn + t * a.qt;
            (key ? ks : qs)[row] = row < a.dk ? to_f32(p[row]) : 0.f;
        }
        float v[V];
        const TIn* vp = static_cast<const TIn*>(a.v) + n * a.vn + t * a.vt + c;
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = in ? to_f32(vp[j]) : 0.f;
        const float decay = a.gate ? expf(log_decay(gate_value(a.gate, n * a.T + t, a.gate_f32), a.form)) : 1.f;
        const float b = gate_value(a.beta, n * a.T + t, a.gate_f32);
        __syncthreads();
        float sum[2 * V + 1];
#pragma unroll
        for (int j = 0; j < 2 * V + 1; ++j) sum[j] = 0.f;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const float k = ks[i * RG + rg], q = qs[i * RG + rg];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                sum[j] = fmaf(k, S[i][j], sum[j]);
                sum[V + j] = fmaf(q, S[i][j], sum[V + j]);
            }
            sum[2 * V] = fmaf(k, q, sum[2 * V]);
        }
#pragma unroll
        for (int j = 0; j < 2 * V + 1; ++j) sum[j] += __shfl_xor(sum[j], 32);
        if ((threadIdx.x & 32) == 0) {
#pragma unroll
            for (int j = 0; j < 2 * V + 1; ++j) sums[wave][cl][j] = sum[j];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2 * V + 1; ++j)
            sum[j] = (sums[0][cl][j] + sums[1][cl][j]) + (sums[2][cl][j] + sums[3][cl][j]);
        float e[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            e[j] = b * fmaf(-decay, sum[j], v[j]);
            const float o = a.scale * fmaf(decay, sum[V + j], sum[2 * V] * e[j]);
            if (in && rg == 0) store_val(op + t * a.dv + j, o);
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const float k = ks[i * RG + rg];
#pragma unroll
            for (int j = 0; j < V; ++j) S[i][j] = fmaf(k, e[j], decay * S[i][j]);
        }
        __syncthreads();  // ks, qs and sums are free again
    }
    if (!in) return;
    for (int64_t t = len + rg; t < a.T; t += RG)
#pragma unroll
        for (int j = 0; j < V; ++j) store_val(op + t * a.dv + j, 0.f);
    if (!a.final_state) return;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int row = i * RG + rg;
        if (row >= a.dk) continue;
        float* p = a.final_state + (n * a.dk + row) * a.dv + c;
        if constexpr (V == 4)
            *reinterpret_cast<float4*>(p) = make_float4(S[i][0], S[i][1], S[i][2], S[i][3]);
        else
            *p = S[i][0];
    }
}

template <typename TIn, int DK, bool kVec, bool kVecV>
hipError_t launch_chunks(const DeltaRule& r, const DeltaArgs& a, hipStream_t stream) {
    constexpr int solve = solve_lds_bytes<TIn, DK>();
    using L = WalkLds<TIn, DK, kOutputs>;
    using Maps = WalkLds<TIn, DK, kMaps>;
    constexpr int walk = L::kBuffers * L::kBytes, maps = Maps::kBuffers * Maps::kBytes;
    static_assert(walk == WalkLds<TIn, DK, kRecording>::kBuffers * WalkLds<TIn, DK, kRecording>::kBytes);
    static_assert(solve <= kGfx950LdsBytes && walk <= kGfx950LdsBytes, "gfx950 gives a workgroup at most 160 KB of LDS");
    delta_solve_kernel<TIn, DK, kVec><<<unsigned(r.N * a.chunks), kThreads, solve, stream>>>(a);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    const unsigned blocks = (r.dv + 63) / 64;
    auto grid = [&](int64_t streams, unsigned each) { return unsigned((streams + 7) / 8 * 8 * each); };
    if (a.segs > 1) {
        delta_chunk_kernel<TIn, DK, kVec, kVecV, kMaps>
            <<<grid(r.N * (a.segs - 1), blocks + (r.dk + 63) / 64), kThreads, maps, stream>>>(a);
        launch_join<DK, false>(r, a, stream);
    }
    if (a.st)
        delta_chunk_kernel<TIn, DK, kVec, kVecV, kRecording><<<grid(r.N * a.segs, blocks), kThreads, walk, stream>>>(a);
    else
        delta_chunk_kernel<TIn, DK, kVec, kVecV, kOutputs><<<grid(r.N * a.segs, blocks), kThreads, walk, stream>>>(a);
    return hipGetLastError();
}

template <typename TIn, bool kVec, bool kVecV>
hipError_t launch_by_width(const DeltaRule& r, const DeltaArgs& a, hipStream_t stream) {
    return r.dk <= 64 ? launch_chunks<TIn, 64, kVec, kVecV>(r, a, stream) : launch_chunks<TIn, 128, kVec, kVecV>(r, a, stream);
}

// Keys by pieces where only the values cannot be: 128 streams of 2048 bf16 tokens, 64 x 50,
// forward and backward 620 -> 525 us, of fp32 ones, 128 x 17, 1480 -> 1307.
template <typename TIn>
hipError_t launch_by_pieces(const DeltaRule& r, const DeltaArgs& a, hipStream_t stream) {
    if (!a.vec_k) return launch_by_width<TIn, false, false>(r, a, stream);
    return a.vec_v && a.vec_o ? launch_by_width<TIn, true, true>(r, a, stream) : launch_by_width<TIn, true, false>(r, a, stream);
}

template <typename TIn, int V>
void launch_step(const DeltaRule& r, const DeltaArgs& a, hipStream_t stream) {
    const dim3 grid(unsigned((r.dv + 32 * V - 1) / (32 * V)), unsigned(r.N));
    if (r.dk <= 64)
        delta_step_kernel<TIn, V, 8><<<grid, kThreads, 0, stream>>>(a);
    else
        delta_step_kernel<TIn, V, 16><<<grid, kThreads, 0, stream>>>(a);
}

}  // namespace

// Chunks of a segment.  One walk has (dv + 63) / 64 workgroups a stream; a chunk takes
// it about 4 us however few there are.  Split, every segment is walked twice, the
// first time with dk columns more and without outputs, so a split pays where it
// makes at least three segments (16 bf16 streams, 128 x 128, of 9 chunks in one 36 us, in
// three 38; of 12 in one 47, in three 46); it aims for a workgroup a CU.
// 16 streams of 32768 tokens, 128 x 128: one walk 1749 us; maps 329, join 28 and walks 298.
// A segment has 4 chunks at least: the join takes a step a segment.  24 ragged fp32
// streams of at most 24 chunks, 64 x 64, forward and backward, segments of 8 94 + 129
// us, of 4 59 + 85, of 3 61 + 77; 16 bf16 ones of 24, 128 x 128, 68, 62, 63.
int64_t delta_segment_chunks(const DeltaRule& r) {
    const int64_t chunks = delta_chunks(r), walks = r.N * ((r.dv + 63) / 64);
    const int64_t segs = std::min<int64_t>(walks > 0 ? 256 / walks : 1, chunks / 4);
    return segs < 3 ? std::max<int64_t>(chunks, 1) : (chunks + segs - 1) / segs;
}

int64_t delta_chunks(const DeltaRule& r) { return (r.T + kChunk - 1) / kChunk; }

DeltaLayout delta_layout(const DeltaRule& r) {
    const int64_t nc = r.N * delta_chunks(r), dvp = (r.dv + 15) / 16 * 16;
    DeltaLayout l;
    const int64_t square = r.dtype == RACE_BF16 ? SquareOf<bf16_t>::kBytes : SquareOf<float>::kBytes;
    l.mm = round256(nc * square);
    l.vec = l.mm + round256(nc * square);
    l.solve_bytes = l.vec + round256(nc * 512);
    const int64_t each = delta_segment_chunks(r), segs = std::max<int64_t>((delta_chunks(r) + each - 1) / each, 1);
    l.segs = int(segs), l.seg_chunks = int(each);
    l.starts = segs > 1 ? round256(r.N * segs * r.dk * r.dk * 4) : 0;
    l.map_x = l.starts + round256(r.N * segs * r.dk * r.dv * 4);
    l.map_bytes = segs > 1 ? l.map_x + round256(r.N * segs * r.dk * r.dv * 4) : 0;
    l.yt = l.solve_bytes + round256(nc * dvp * dk_padded(r) * 4);
    l.map_a = l.yt + round256(nc * dvp * kChunk * 4);
    l.record_bytes = l.map_a + l.starts;
    return l;
}

hipError_t launch_delta(const DeltaRule& r, const DeltaInputs& in, const float* state, void* out, float* final_state,
                        void* records, void* workspace, hipStream_t stream) {
    DeltaArgs a = delta_args(r, in);
    a.state = state, a.out = out, a.final_state = final_state;
    if (!records && r.T <= kDeltaStepTokens) {
        const bool four = r.dv % 4 == 0;
        if (r.dtype == RACE_BF16)
            four ? launch_step<bf16_t, 4>(r, a, stream) : launch_step<bf16_t, 1>(r, a, stream);
        else
            four ? launch_step<float, 4>(r, a, stream) : launch_step<float, 1>(r, a, stream);
        return hipGetLastError();
    }
    const DeltaLayout l = delta_layout(r);
    unsigned char* maps = static_cast<unsigned char*>(workspace);
    unsigned char* base = records ? static_cast<unsigned char*>(records) : maps + l.map_bytes;
    a.tm = base, a.mm = base + l.mm;
    a.vec = reinterpret_cast<float*>(base + l.vec);
    if (records) a.st = reinterpret_cast<float*>(base + l.solve_bytes), a.yt = reinterpret_cast<float*>(base + l.yt);
    a.segs = l.segs, a.seg_chunks = l.seg_chunks;
    if (l.segs > 1) {
        a.map_a = reinterpret_cast<float*>(records ? base + l.map_a : maps);
        a.starts = reinterpret_cast<float*>(maps + l.starts), a.map_x = reinterpret_cast<float*>(maps + l.map_x);
    }
    return r.dtype == RACE_BF16 ? launch_by_pieces<bf16_t>(r, a, stream) : launch_by_pieces<float>(r, a, stream);
}

}  // namespace race
