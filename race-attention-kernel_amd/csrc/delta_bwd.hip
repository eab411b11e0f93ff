// delta_bwd.hip -- the gated delta rule, backward.  With delta_chunk.hip's names
// for a chunk, M = scale Gam o Q K^T b, and dS' the gradient of the state behind it:
//
//     dY = M^T dO + Z b (K dS'),   dD = T^T dY = dV,
//     dS = e^{G_last} dS' + scale Q^T (E dO) - K^T (E dD)
//
// runs backward from chunk to chunk (delta_bwd_walk_kernel), 16 columns of dS in a
// wave's registers as the forward's S.  Then every chunk by itself
// (delta_grads_kernel), from the kept S, Y and the walk's dS', dD, with
// P = scale dO Y^T, H = dD Y^T, L_ij = Gam_ij b_j P_ij (j <= i),
// X_ij = -Gam_ij b_j H_ij (j < i):
//
//     dQ = scale E (dO S^T) + L K
//     dK = L^T Q + (X + X^T) K + Z b (Y dS'^T) - E (dD S^T)
//     db_j = sum_i Gam_ij (q_i.k_j P_ij - k_i.k_j H_ij) + Z_j k_j.(dS' Y_j)
//     dG_i = E_i (scale q_i.(S dO_i) - k_i.(S dD_i)) + R_i - C_i - c_i,
//
// R and C the row and column sums of L_ij q_i.k_j + X_ij k_i.k_j, c_i = b_i Z_i
// k_i.(dS' Y_i), and dG_last more by sum c + e^{G_last} <S, dS'>; a log decay's
// gradient is the sum of the dG from it on.  Pairs of tokens that a decay does not
// lie between cancel in it exactly, R and C holding the same numbers.
//
// Bound by memory: the walk's and the forward's kept states.  Key streams that
// several value streams share sum their gradients in the registers of one
// workgroup, in order: results are bitwise reproducible.
#include "delta_tiles.h"

namespace race {
namespace {

using namespace delta;

struct DeltaBwdArgs {
    DeltaArgs f;
    const void* dout;
    const float* dfinal;
    void *ds, *dd;  // [N][chunks][dvp] columns of dS' [DK] and dD [64]
    void *dq, *dk, *dv, *dgate, *dbeta;
    float* dstate;
};

// ---- the walk ----

template <typename TIn, int DK, bool kVec>
__global__ __launch_bounds__(kThreads) void delta_bwd_walk_kernel(const DeltaBwdArgs w) {
    extern __shared__ __align__(16) unsigned char lds[];
    const DeltaArgs& a = w.f;
    using L = ChunkLds<TIn, DK>;  // dO in the place of V
    using Rows = Tile<TIn, DK>;
    using Square = Tile<TIn, 64>;
    using One = OneT<TIn>;
    using Two = TwoT<TIn>;
    constexpr int NS = DK / 32;
    int64_t n;
    int cb;
    if (!stream_and_block(a.N, (a.dv + 63) / 64, n, cb)) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, lr = lane & 15;
    const bool odd = g & 1;
    const int c0 = cb * 64 + wave * 16, col = c0 + lr;
    const bool active = c0 < a.dv;
    const int64_t nk = n / a.group, len = a.live.of(n, a.T);
    const int chunks = int((len + kChunk - 1) / kChunk);
    const TIn* kp = static_cast<const TIn*>(a.k) + nk * a.kn;
    const TIn* qp = static_cast<const TIn*>(a.q) + nk * a.qn;
    const TIn* op = static_cast<const TIn*>(w.dout) + n * a.T * a.dv + cb * 64;

    f32x4 dS[DK / 16];
#pragma unroll
    for (int i = 0; i < DK / 16; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = tok(i, 4 * g + r);
            dS[i][r] = w.dfinal && active && row < a.dk && col < a.dv ? w.dfinal[(n * a.dk + row) * a.dv + col] : 0.f;
        }

    Stage<TIn, DK, kThreads, kVec> sk, sq;
    StageDense<TIn, 64, kTwoRows<TIn>, kThreads> stm;
    StageDense<TIn, 64, kChunk, kThreads> smm;
    Stage<TIn, 64, kThreads, kVec> so;
    float svec;
    sk.init(a.kt, a.dk);
    sq.init(a.qt, a.dk);
    so.init(a.dv, a.dv - cb * 64);
    auto fetch = [&](int c, int part) {  // as the forward's
        const int64_t nc = n * a.chunks + c, t0 = int64_t(c) * kChunk;
        const int live = int(len - t0 < kChunk ? len - t0 : kChunk);
        if (part == 0) sk.load(kp + t0 * a.kt, a.kt, live, a.dk);
        if (part == 1) sq.load(qp + t0 * a.qt, a.qt, live, a.dk);
        if (part == 2) stm.load(static_cast<const TIn*>(a.tm) + nc * (kTwoRows<TIn> * kChunk));
        if (part == 3) {
            smm.load(static_cast<const TIn*>(a.mm) + nc * (kChunk * kChunk));
            so.load(op + t0 * a.dv, a.dv, live, a.dv - cb * 64);
            svec = a.vec[nc * 128 + (threadIdx.x & 127)];
        }
    };
    // What a lane adds to a tile's start.
    const int k_row = Rows::row_base(lr, g), k_col = Rows::column_base(lr, g), s_col = Square::column_base(lr, g);
    const int o_at = Square::block_base(16 * wave, lr, g);
    if (chunks > 0)
        for (int p = 0; p < 4; ++p) fetch(chunks - 1, p);
    for (int c = chunks - 1; c >= 0; --c) {
        unsigned char* buf = lds + (L::kBuffers == 2 ? (c & 1) * L::kBytes : 0);
        if (L::kBuffers == 1 && c < chunks - 1) __syncthreads();  // the chunk before is done with the buffer
        sk.put(buf + L::kK);
        sq.put(buf + L::kQ);
        stm.put(buf + L::kT);
        smm.put(buf + L::kM);
        so.put(buf + L::kV);
        reinterpret_cast<float*>(buf + L::kVec)[threadIdx.x & 127] = svec;
        const int next = c > 0 ? c - 1 : 0;  // the last chunk's loads are not used
        __syncthreads();
        if (!active) {
            for (int p = 0; p < 4; ++p) fetch(next, p);
            continue;
        }
        const float* E = reinterpret_cast<const float*>(buf + L::kVec);
        const int64_t nc = n * a.chunks + c;
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
        One kf[NS][4];
        f32x4 o[4], e[4];
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int b = 0; b < 4; ++b) kf[i][b] = Rows::one(buf + L::kK, k_row, b, i);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            o[b] = Square::block(buf + L::kV, o_at, b);
            e[b] = *reinterpret_cast<const f32x4*>(E + tok(b, 4 * g));
        }
        Two s[NS];
        TIn* ds = static_cast<TIn*>(w.ds) + (nc * a.dvp + col) * DK + 8 * g;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            operand(dS[2 * i], dS[2 * i + 1], odd, s[i]);
            store_run(ds + 32 * i, delta::first(s[i]));
        }
        stage_wall();
        fetch(next, 0);
        One mf[4], mg[2];
        f32x4 zb[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            mf[b] = Square::transposed(buf + L::kM, s_col, 1, b);
            zb[b] = *reinterpret_cast<const f32x4*>(E + 64 + tok(b, 4 * g));
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) mg[b] = Square::transposed(buf + L::kM, s_col, 0, b);
        // dO as it is, and as E dO scale.
        One od[2], eo[2];
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            operand(o[2 * kk], o[2 * kk + 1], odd, od[kk]);
            operand(o[2 * kk] * e[2 * kk] * a.scale, o[2 * kk + 1] * e[2 * kk + 1] * a.scale, odd, eo[kk]);
        }
        // dY = M^T dO + Z b (K dS').
        f32x4 x[4];
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int b = 0; b < 4; ++b) x[b] = mac(kf[i][b], s[i], i == 0 ? zero : x[b]);
        stage_wall();
        fetch(next, 1);
        Two tf[4], tg[2];
#pragma unroll
        for (int b = 0; b < 4; ++b) tf[b] = Square::transposed_two(buf + L::kT, s_col, 1, b);
#pragma unroll
        for (int b = 0; b < 2; ++b) tg[b] = Square::transposed_two(buf + L::kT, s_col, 0, b);
#pragma unroll
        for (int b = 0; b < 4; ++b) x[b] = mac(mf[b], od[1], x[b] * zb[b]);
#pragma unroll
        for (int b = 0; b < 2; ++b) x[b] = mac(mg[b], od[0], x[b]);
        Two y[2];
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) operand(x[2 * kk], x[2 * kk + 1], odd, y[kk]);
        stage_wall();
        fetch(next, 2);
        One qc[2][DK / 16];
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
            for (int i = 0; i < DK / 16; ++i) qc[kk][i] = Rows::transposed(buf + L::kQ, k_col, kk, i);
        // dD = T^T dY.
#pragma unroll
        for (int b = 0; b < 4; ++b) x[b] = mac(tf[b], y[1], zero);
#pragma unroll
        for (int b = 0; b < 2; ++b) x[b] = mac(tg[b], y[0], x[b]);
        stage_wall();
        fetch(next, 3);
        One kc[2][DK / 16];
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
            for (int i = 0; i < DK / 16; ++i) kc[kk][i] = Rows::transposed(buf + L::kK, k_col, kk, i);
        // dS = e^{G_last} dS' + scale Q^T (E dO) - K^T (E dD).
        const float decay = E[63];
#pragma unroll
        for (int i = 0; i < DK / 16; ++i) dS[i] *= decay;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
            for (int i = 0; i < DK / 16; ++i) dS[i] = mac(qc[kk][i], eo[kk], dS[i]);
        Two d[2];
        TIn* dd = static_cast<TIn*>(w.dd) + (nc * a.dvp + col) * kChunk + 8 * g;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            One plain;
            operand(x[2 * kk], x[2 * kk + 1], odd, plain);
            store_run(dd + 32 * kk, plain);
            operand(x[2 * kk] * -e[2 * kk], x[2 * kk + 1] * -e[2 * kk + 1], odd, d[kk]);
        }
        stage_wall();
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
            for (int i = 0; i < DK / 16; ++i) dS[i] = mac(kc[kk][i], d[kk], dS[i]);
    }
    if (!w.dstate || !active || col >= a.dv) return;
#pragma unroll
    for (int i = 0; i < DK / 16; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = tok(i, 4 * g + r);
            if (row < a.dk) w.dstate[(n * a.dk + row) * a.dv + col] = dS[i][r];
        }
}

// ---- the chunks' gradients ----

constexpr int kGradThreads = 512;

// Columns of the state a step takes: 64 of bf16, 32 of fp32 for the LDS.
template <typename TIn>
constexpr int kSlice = sizeof(TIn) == 2 ? 64 : 32;

template <typename TIn, int DK>
struct GradLds {
    static constexpr int SL = kSlice<TIn>, kS = int(sizeof(TIn));
    static constexpr int kK = 0, kQ = Tile<TIn, DK>::kBytes, kSt = 2 * kQ, kDs = kSt + SL * DK * kS;
    static constexpr int kSquare = Tile<TIn, 64>::kBytes;
    // L^T and X^T lie over the slices of S and dS', once those are read.
    static constexpr int kL = kSt, kX = kSt + kSquare;
    static constexpr int kStates = 2 * SL * DK * kS > 2 * kSquare ? 2 * SL * DK * kS : 2 * kSquare;
    static constexpr int kYt = kSt + kStates, kDd = kYt + SL * kChunk * kS, kO = kDd + SL * kChunk * kS;
    static constexpr int kBytes = kO + kChunk * SL * kS;
};

// Dense rows of K values to a tile, zeros past the first `rows` of ROWS.
template <typename E, int K, int ROWS>
__device__ __forceinline__ void stage_rows(const E* p, int rows, unsigned char* t) {
    constexpr int kChunks = Tile<E, K>::kChunks;
#pragma unroll
    for (int i = 0; i < (ROWS * kChunks + kGradThreads - 1) / kGradThreads; ++i) {
        const int q = int(threadIdx.x) + i * kGradThreads, row = q / kChunks, u = q % kChunks;
        if (ROWS * kChunks % kGradThreads != 0 && q >= ROWS * kChunks) break;
        const uint4 x = row < rows ? reinterpret_cast<const uint4*>(p)[q] : make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(t + Tile<E, K>::at(row, u)) = x;
    }
}

template <typename TIn>
__device__ __forceinline__ float dot16(const uint4& x, const uint4& y, float s) {
#pragma unroll
    for (int i = 0; i < 16 / int(sizeof(TIn)); ++i) s = fmaf(mfma::Elem<TIn>::get(x, i), mfma::Elem<TIn>::get(y, i), s);
    return s;
}

__device__ __forceinline__ void store_gate(void* p, int64_t i, int f32, float x) {
    if (f32)
        static_cast<float*>(p)[i] = x;
    else
        static_cast<bf16_t*>(p)[i] = f32_to_bf16(x);
}

// A chunk of a key stream: eight waves, wave (th, dq) of 32 tokens and a quarter of
// the key columns; of the 64 x 64 matrices 32 rows and 16 columns.
template <typename TIn, int DK, bool kVec>
__global__ __launch_bounds__(kGradThreads) void delta_grads_kernel(const DeltaBwdArgs w) {
    extern __shared__ __align__(16) unsigned char lds[];
    __shared__ double G[kChunk];
    __shared__ float beta[kChunk];
    __shared__ float row_sum[4][kChunk], col_sum[2][kChunk], b_sum[2][kChunk], dots[3][4][kChunk], ss[8];
    const DeltaArgs& a = w.f;
    using L = GradLds<TIn, DK>;
    using Rows = Tile<TIn, DK>;
    using Square = Tile<TIn, 64>;
    using Out = Tile<TIn, L::SL>;
    using One = OneT<TIn>;
    constexpr int NB = DK / 64, SL = L::SL;
    const int64_t nkc = blockIdx.x, nk = nkc / a.chunks;
    const int c = int(nkc - nk * a.chunks), t0 = c * kChunk;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, lr = lane & 15;
    const int th = wave >> 2, dq = wave & 3;
    const int here = int(a.T - t0 < kChunk ? a.T - t0 : kChunk);  // rows of the chunk, live or not
    int most = 0;
    for (int h = 0; h < a.group; ++h) {
        const int64_t l = a.live.of(nk * a.group + h, a.T) - t0;
        most = max(most, int(l < kChunk ? l : kChunk));
    }
    if (most > 0) {
        Stage<TIn, DK, kGradThreads, kVec> sk, sq;
        sk.init(a.kt, a.dk);
        sq.init(a.qt, a.dk);
        sk.load(static_cast<const TIn*>(a.k) + nk * a.kn + t0 * a.kt, a.kt, most, a.dk);
        sq.load(static_cast<const TIn*>(a.q) + nk * a.qn + t0 * a.qt, a.qt, most, a.dk);
        sk.put(lds + L::kK);
        sq.put(lds + L::kQ);
    }
    const int k_col = Rows::column_base(lr, g), s_col = Square::column_base(lr, g), o_row = Out::row_base(lr, g);
    const int k_row = Rows::row_base(lr, g), s_row = Square::row_base(lr, g);
    f32x4 gq[2][NB], gk[2][NB];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int b = 0; b < NB; ++b) gq[i][b] = gk[i][b] = f32x4{0.f, 0.f, 0.f, 0.f};

    for (int h = 0; h < a.group; ++h) {
        const int64_t n = nk * a.group + h, len = a.live.of(n, a.T), nc = n * a.chunks + c;
        const int live = int(len - t0 < kChunk ? len - t0 : kChunk);
        TIn* dv = w.dv ? static_cast<TIn*>(w.dv) + (n * a.T + t0) * a.dv : nullptr;
        if (live <= 0) {
            if (dv)
                for (int i = threadIdx.x; i < here * a.dv; i += kGradThreads) store_val(dv + i, 0.f);
            if (int(threadIdx.x) < here) {
                if (w.dgate) store_gate(w.dgate, n * a.T + t0 + threadIdx.x, a.gate_f32, 0.f);
                if (w.dbeta) store_gate(w.dbeta, n * a.T + t0 + threadIdx.x, a.gate_f32, 0.f);
            }
            continue;
        }
        __syncthreads();  // K and Q are there; the stream before is done with the tiles and the sums
        if (wave == 0) {
            const int64_t at = n * a.T + t0 + lane;
            double s = lane < live && a.gate ? double(log_decay(gate_value(a.gate, at, a.gate_f32), a.form)) * kLog2e : 0.0;
            for (int d = 1; d < 64; d <<= 1) {
                const double o = __shfl_up(s, d);
                if (lane >= d) s += o;
            }
            G[lane] = s;
            beta[lane] = lane < live ? gate_value(a.beta, at, a.gate_f32) : 0.f;
        }
        f32x4 P[2], H[2], qs[2][NB], fs[2][NB], zs[2][NB];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            P[i] = H[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int b = 0; b < NB; ++b) qs[i][b] = fs[i][b] = zs[i][b] = P[i];
        }
        float s_ds = 0.f;
        for (int v0 = 0; v0 < a.dv; v0 += SL) {
            if (v0 > 0) __syncthreads();  // the slice before is read
            const int rows = min(SL, a.dvp - v0);
            {
                constexpr int kCk = Rows::kChunks;
                const uint4* sp = reinterpret_cast<const uint4*>(static_cast<const TIn*>(a.st) + (nc * a.dvp + v0) * DK);
                const uint4* dp = reinterpret_cast<const uint4*>(static_cast<const TIn*>(w.ds) + (nc * a.dvp + v0) * DK);
#pragma unroll
                for (int i = 0; i < SL * kCk / kGradThreads; ++i) {
                    const int q = int(threadIdx.x) + i * kGradThreads, row = q / kCk, u = q % kCk;
                    uint4 x = make_uint4(0, 0, 0, 0), y = x;
                    if (row < rows) x = sp[q], y = dp[q];
                    s_ds = dot16<TIn>(x, y, s_ds);
                    *reinterpret_cast<uint4*>(lds + L::kSt + Rows::at(row, u)) = x;
                    *reinterpret_cast<uint4*>(lds + L::kDs + Rows::at(row, u)) = y;
                }
            }
            stage_rows<TIn, 64, SL>(static_cast<const TIn*>(a.yt) + (nc * a.dvp + v0) * kChunk, rows, lds + L::kYt);
            stage_rows<TIn, 64, SL>(static_cast<const TIn*>(w.dd) + (nc * a.dvp + v0) * kChunk, rows, lds + L::kDd);
            {
                const TIn* p = static_cast<const TIn*>(w.dout) + (n * a.T + t0) * a.dv + v0;
                constexpr int kEights = SL / 8, kVecs = Eight<TIn>::kVecs;
                const auto view = mfma::make_rsrc(p, ((live - 1) * int64_t(a.dv) + a.dv - v0) * int(sizeof(TIn)));
#pragma unroll
                for (int i = 0; i < (kChunk * kEights + kGradThreads - 1) / kGradThreads; ++i) {
                    const int q = int(threadIdx.x) + i * kGradThreads, row = q / kEights, u = q % kEights;
                    if (kChunk * kEights < kGradThreads && q >= kChunk * kEights) break;
                    Eight<TIn> x;
                    if constexpr (kVec) {
#pragma unroll
                        for (int j = 0; j < kVecs; ++j)
                            x.v[j] = mfma::buf_load16<mfma::kPolicyDefault>(view, piece_at<TIn>(row, a.dv, 8 * u + 4 * j, a.dv - v0));
                    } else {
                        x.load(p + row * a.dv + 8 * u, row < live ? a.dv - v0 - 8 * u : 0);
                    }
#pragma unroll
                    for (int j = 0; j < kVecs; ++j)
                        *reinterpret_cast<uint4*>(lds + L::kO + Out::at(row, kVecs * u + j)) = x.v[j];
                }
            }
            __syncthreads();
#pragma unroll
            for (int kk = 0; kk < SL / 32; ++kk) {
                const One yc = Square::transposed(lds + L::kYt, s_col, kk, dq);
                One ya[2], da[2], oa[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int b = 2 * th + i;
                    ya[i] = Square::transposed(lds + L::kYt, s_col, kk, b);
                    da[i] = Square::transposed(lds + L::kDd, s_col, kk, b);
                    oa[i] = Out::one(lds + L::kO, o_row, b, kk);
                    P[i] = mac(oa[i], yc, P[i]);
                    H[i] = mac(da[i], yc, H[i]);
                    // A token's dV: these waves hold the same rows, each writes every fourth run.
                    if (dv && ((v0 >> 5) + kk) % 4 == dq && tok(b, lr) < here) {
                        const int cv = v0 + 32 * kk + 8 * g;
                        TIn* o = dv + int64_t(tok(b, lr)) * a.dv + cv;
                        if (kVec && cv + 8 <= a.dv) {
                            store_run(o, da[i]);
                        } else {
                            const auto run = __builtin_bit_cast(Eight<TIn>, da[i]);
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                constexpr int kPer = 16 / int(sizeof(TIn));
                                if (cv + e < a.dv) store_val(o + e, mfma::Elem<TIn>::get(run.v[e / kPer], e % kPer));
                            }
                        }
                    }
                }
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const One st = Rows::transposed(lds + L::kSt, k_col, kk, dq * NB + b);
                    const One ds = Rows::transposed(lds + L::kDs, k_col, kk, dq * NB + b);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        qs[i][b] = mac(st, oa[i], qs[i][b]);
                        fs[i][b] = mac(st, da[i], fs[i][b]);
                        zs[i][b] = mac(ds, ya[i], zs[i][b]);
                    }
                }
            }
        }
        // Rows tok(2 th + i, 4 g + r), column tok(dq, lr) of the 64 x 64 matrices.
        const int jc = tok(dq, lr);
        const float bj = beta[jc];
        const double Gj = G[jc];
        float in_row[2][4], in_col = 0.f, in_b = 0.f;
        f32x4 Lm[2], Xm[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            f32x4 qk = {0.f, 0.f, 0.f, 0.f}, kk = qk;
#pragma unroll
            for (int s = 0; s < DK / 32; ++s) {
                const One kj = Rows::one(lds + L::kK, k_row, dq, s);
                qk = mac(Rows::one(lds + L::kQ, k_row, 2 * th + i, s), kj, qk);
                kk = mac(Rows::one(lds + L::kK, k_row, 2 * th + i, s), kj, kk);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = tok(2 * th + i, 4 * g + r);
                const float e = row >= jc ? __builtin_amdgcn_exp2f(float(G[row] - Gj)) : 0.f;
                const float p = a.scale * e * P[i][r], hm = row > jc ? -e * H[i][r] : 0.f;
                Lm[i][r] = bj * p;
                Xm[i][r] = bj * hm;
                const float pair = fmaf(p, qk[r], hm * kk[r]);
                in_b += pair;
                in_row[i][r] = bj * pair;
                in_col += bj * pair;
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
#pragma unroll
                for (int d = 1; d < 16; d <<= 1) in_row[i][r] += __shfl_xor(in_row[i][r], d);
                if (lr == 0) row_sum[dq][tok(2 * th + i, 4 * g + r)] = in_row[i][r];
            }
        in_col += __shfl_xor(in_col, 16);
        in_col += __shfl_xor(in_col, 32);
        in_b += __shfl_xor(in_b, 16);
        in_b += __shfl_xor(in_b, 32);
        if (g == 0) col_sum[th][jc] = in_col, b_sum[th][jc] = in_b;
        for (int d = 1; d < 64; d <<= 1) s_ds += __shfl_xor(s_ds, d);
        if (lane == 0) ss[wave] = s_ds;
        // What comes from the states, by rows: a token a lane, its key columns in registers.
        const double last = G[63];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = tok(2 * th + i, lr);
            const float e = __builtin_amdgcn_exp2f(float(G[row])), z = __builtin_amdgcn_exp2f(float(last - G[row]));
            float dot[3] = {0.f, 0.f, 0.f};
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int cd = tok(dq * NB + b, 4 * g);
                const int at = Rows::four_at(row, cd);
                const f32x4 q4 = Rows::four(lds + L::kQ, at), k4 = Rows::four(lds + L::kK, at);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float qv = qs[i][b][r] * (e * a.scale), fv = fs[i][b][r] * e, zv = zs[i][b][r] * z;
                    dot[0] = fmaf(q4[r], qv, dot[0]);
                    dot[1] = fmaf(k4[r], fv, dot[1]);
                    dot[2] = fmaf(k4[r], zv, dot[2]);
                    gq[i][b][r] += qv;
                    gk[i][b][r] += beta[row] * zv - fv;
                }
            }
#pragma unroll
            for (int x = 0; x < 3; ++x) {
                dot[x] += __shfl_xor(dot[x], 16);
                dot[x] += __shfl_xor(dot[x], 32);
                if (g == 0) dots[x][dq][row] = dot[x];
            }
        }
        __syncthreads();  // the slices of S and dS' are read
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int at = Square::four_at(jc, tok(2 * th + i, 4 * g));
            Square::put4(lds + L::kL, at, Lm[i]);
            Square::put4(lds + L::kX, at, Xm[i]);
        }
        __syncthreads();
        if (wave == 0 && (w.dgate || w.dbeta)) {
            const float z = dots[2][0][lane] + dots[2][1][lane] + dots[2][2][lane] + dots[2][3][lane];
            const int64_t at = n * a.T + t0 + lane;
            if (w.dbeta && lane < here)
                store_gate(w.dbeta, at, a.gate_f32, lane < live ? b_sum[0][lane] + b_sum[1][lane] + z : 0.f);
            if (w.dgate) {
                const float bz = beta[lane] * z;
                double all = bz;
                for (int d = 1; d < 64; d <<= 1) all += __shfl_xor(all, d);
                float s = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) s += ss[i];
                double dg = -double(bz);
#pragma unroll
                for (int x = 0; x < 4; ++x) dg += double(row_sum[x][lane]) + dots[0][x][lane] - dots[1][x][lane];
                dg -= double(col_sum[0][lane]) + col_sum[1][lane];
                if (lane == 63) dg += all + double(__builtin_amdgcn_exp2f(float(last))) * s;
                for (int d = 1; d < 64; d <<= 1) {
                    const double o = __shfl_down(dg, d);
                    if (lane + d < 64) dg += o;
                }
                float x = 0.f;
                if (lane < live) {
                    const float gv = gate_value(a.gate, at, a.gate_f32);
                    const bool lowest = log_decay(gv, a.form) <= kLowestLog;  // constant there
                    x = lowest ? 0.f : float(dg);
                    if (a.form == RACE_GATE_SIGMOID) x *= 1.f / (1.f + expf(gv));
                }
                if (lane < here) store_gate(w.dgate, at, a.gate_f32, x);
            }
        }
        // dQ += L K, dK += L^T Q + (X + X^T) K; a token a lane as above.
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int b = 2 * th + i;
                One l, lt, x, xt;
                if (kk <= th) {
                    l = Square::transposed(lds + L::kL, s_col, kk, b);
                    x = Square::transposed(lds + L::kX, s_col, kk, b);
                }
                if (kk >= th) {
                    lt = Square::one(lds + L::kL, s_row, b, kk);
                    xt = Square::one(lds + L::kX, s_row, b, kk);
                }
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    const One kf = Rows::transposed(lds + L::kK, k_col, kk, dq * NB + nb);
                    if (kk <= th) {
                        gq[i][nb] = mac(kf, l, gq[i][nb]);
                        gk[i][nb] = mac(kf, x, gk[i][nb]);
                    }
                    if (kk >= th) {
                        gk[i][nb] = mac(kf, xt, gk[i][nb]);
                        gk[i][nb] = mac(Rows::transposed(lds + L::kQ, k_col, kk, dq * NB + nb), lt, gk[i][nb]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int row = tok(2 * th + i, lr);
        if (row >= here) continue;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int cd = tok(dq * NB + b, 4 * g), there = a.dk - cd;
            if (there <= 0) continue;
            const int64_t at = (nk * a.T + t0 + row) * a.dk + cd;
            for (int x = 0; x < 2; ++x) {
                TIn* p = static_cast<TIn*>(x ? w.dk : w.dq);
                if (!p) continue;
                const f32x4 v = x ? gk[i][b] : gq[i][b];
                if (a.dk % 4 == 0) {
                    store4_of(p + at, v);
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (r < there) store_val(p + at + r, v[r]);
                }
            }
        }
    }
}

template <typename TIn, int DK, bool kVec>
hipError_t launch_backward(const DeltaRule& r, const DeltaBwdArgs& w, hipStream_t stream) {
    using L = ChunkLds<TIn, DK>;
    constexpr int walk = L::kBuffers * L::kBytes, grads = GradLds<TIn, DK>::kBytes;
    static_assert(walk <= kGfx950LdsBytes && grads + 8192 <= kGfx950LdsBytes, "gfx950 gives a workgroup at most 160 KB of LDS");
    const int64_t blocks = (r.dv + 63) / 64;
    delta_bwd_walk_kernel<TIn, DK, kVec><<<unsigned((r.N + 7) / 8 * 8 * blocks), kThreads, walk, stream>>>(w);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    if (!w.dq && !w.dk && !w.dv && !w.dgate && !w.dbeta) return hipSuccess;
    delta_grads_kernel<TIn, DK, kVec><<<unsigned(r.Nk * w.f.chunks), kGradThreads, grads, stream>>>(w);
    return hipGetLastError();
}

template <typename TIn, bool kVec>
hipError_t launch_by_width(const DeltaRule& r, const DeltaBwdArgs& w, hipStream_t stream) {
    return r.dk <= 64 ? launch_backward<TIn, 64, kVec>(r, w, stream) : launch_backward<TIn, 128, kVec>(r, w, stream);
}

}  // namespace

int64_t delta_bwd_bytes(const DeltaRule& r) {
    const int64_t nc = r.N * delta_chunks(r), es = r.dtype == RACE_BF16 ? 2 : 4, dvp = (r.dv + 15) / 16 * 16;
    return round256(nc * dvp * dk_padded(r) * es) + round256(nc * dvp * kChunk * es);
}

hipError_t launch_delta_bwd(const DeltaRule& r, const DeltaInputs& in, const void* dout, const float* dfinal,
                            const void* records, const DeltaGrads& g, void* scratch, hipStream_t stream) {
    DeltaBwdArgs w = {};
    w.f = delta_args(r, in);
    const DeltaLayout l = delta_layout(r);
    unsigned char* base = const_cast<unsigned char*>(static_cast<const unsigned char*>(records));
    w.f.tm = base, w.f.mm = base + l.mm, w.f.vec = reinterpret_cast<float*>(base + l.vec);
    w.f.st = base + l.solve_bytes, w.f.yt = base + l.yt;
    w.dout = dout, w.dfinal = dfinal;
    const int64_t es = r.dtype == RACE_BF16 ? 2 : 4;
    w.ds = scratch;
    w.dd = static_cast<unsigned char*>(scratch) + round256(r.N * w.f.chunks * w.f.dvp * dk_padded(r) * es);
    w.dq = g.dq, w.dk = g.dk, w.dv = g.dv, w.dgate = g.dgate, w.dbeta = g.dbeta, w.dstate = g.dstate;
    const bool vec = w.f.vec_k && w.f.vec_o;
    if (r.dtype == RACE_BF16)
        return vec ? launch_by_width<bf16_t, true>(r, w, stream) : launch_by_width<bf16_t, false>(r, w, stream);
    return vec ? launch_by_width<float, true>(r, w, stream) : launch_by_width<float, false>(r, w, stream);
}

}  // namespace race
