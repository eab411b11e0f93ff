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
// Precision as the forward's: sums are fp32, S, Y, dS' and dD are kept in fp32, and bf16 rows'
// products take what is computed in three parts; where every gradient of the second
// launch is rounded to bf16 right away, in two.  (With S, Y, dS', dD, L and X rounded to
// bf16 once each, the gradients were off by twice what their own rounding costs.)
//
// 128 streams of 4096 bf16 tokens, 128 x 128: the walk 395 us, bound as the forward's;
// the gradients 710 us (three parts 845; rounded once 485), whose workgroups stay and load
// the next slice's rows meanwhile: a chunk's kept states come in slices of 32 value
// columns, and its 64 x 64 matrices and sums between two barriers take half of the time.
// Key streams that several value streams share sum their gradients in the registers of one
// workgroup, in order: results are bitwise reproducible.
#include "delta_tiles.h"

namespace race {
namespace {

using namespace delta;

struct DeltaBwdArgs {
    DeltaArgs f;
    const void* dout;
    const float* dfinal;
    float *ds, *dd;  // [N][chunks][dvp] columns of dS' [DK] and dD [64]
    void *dq, *dk, *dv, *dgate, *dbeta;
    float* dstate;
};

// ---- the walk ----

__device__ __forceinline__ void store_gate(void* p, int64_t i, int f32, float x) {
    if (f32)
        static_cast<float*>(p)[i] = x;
    else
        static_cast<bf16_t*>(p)[i] = f32_to_bf16(x);
}

// dO in the place of V.  192 streams of 577 tokens, 64 x 128: two workgroups a CU 73 us, one 86.
template <typename TIn, int DK>
using BwdWalkLds = ChunkLds<TIn, DK, 3, true, !two_a_cu(sizeof(TIn) * DK, false)>;

// kMaps: no records, but what the segment adds to a gradient of zero behind it (the
// last one: to dfinal), to map_x.
template <typename TIn, int DK, bool kVec, bool kVecV, bool kMaps>
__global__ __launch_bounds__(kThreads, two_a_cu(sizeof(TIn) * DK, false) ? 2 : 1) void delta_bwd_walk_kernel(const DeltaBwdArgs w) {
    extern __shared__ __align__(16) unsigned char lds[];
    const DeltaArgs& a = w.f;
    using L = BwdWalkLds<TIn, DK>;
    using Rows = Tile<TIn, DK>;
    using Square = Tile<TIn, 64>;
    using One = OneT<TIn>;
    using Three = ThreeT<TIn>;
    constexpr int NS = DK / 32;
    // M, T and Q are read behind a product, for its registers: 78 -> 73 us in the case above.
    constexpr bool kLate = two_a_cu(sizeof(TIn) * DK, false);
    const int walks = kMaps ? a.segs - 1 : a.segs;  // no gradient goes on before the first segment
    int64_t ns;
    int cb;
    if (!stream_and_block(a.N * walks, (a.dv + 63) / 64, ns, cb)) return;
    const int64_t n = unsigned(ns) / unsigned(walks);
    const int seg = int(ns - n * walks) + (kMaps ? 1 : 0);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, lr = lane & 15;
    const bool odd = g & 1;
    const int c0 = cb * 64 + wave * 16, col = c0 + lr;
    const bool active = c0 < a.dv;
    const int64_t nk = a.key_stream(n), len = a.len_of(n);
    const int all = int((len + kChunk - 1) / kChunk);
    const int from = min(seg * a.seg_chunks, all), chunks = min(from + a.seg_chunks, all);
    const TIn* kp = static_cast<const TIn*>(a.k) + nk * a.kn;
    const TIn* qp = static_cast<const TIn*>(a.q) + nk * a.qn;
    const TIn* op = static_cast<const TIn*>(w.dout) + n * a.T * a.dv + cb * 64;
    const float* behind = !kMaps && a.starts             ? a.starts + ns * a.dk * a.dv
                          : w.dfinal && seg == a.segs - 1 ? w.dfinal + n * a.dk * a.dv
                                                          : nullptr;

    f32x4 dS[DK / 16];
    if (behind) {
        const StateView from(behind, a.dk, a.dv);
#pragma unroll
        for (int i = 0; i < DK / 16; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) dS[i][r] = from.one(tok(i, 4 * g + r), col);
    } else {
#pragma unroll
        for (int i = 0; i < DK / 16; ++i) dS[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    Stage<TIn, DK, kThreads, kVec> sk, sq;
    StageSquare<TIn, 3> stm, smm;
    Stage<TIn, 64, kThreads, kVecV> so;
    float svec;
    sk.init(a.kt, a.dk);
    sq.init(a.qt, a.dk);
    so.init(a.dv, a.dv - cb * 64);
    auto fetch = [&](int c, int part) {  // as the forward's
        const int64_t nc = n * a.chunks + c, t0 = int64_t(c) * kChunk;
        const int live = int(len - t0 < kChunk ? len - t0 : kChunk);
        if (part == 0) sk.load(kp + t0 * a.kt, live);
        if (part == 1) sq.load(qp + t0 * a.qt, live);
        if (part == 2) stm.load(a.tm + nc * SquareOf<TIn>::kBytes);
        if (part == 3) {
            smm.load(a.mm + nc * SquareOf<TIn>::kBytes);
            so.load(op + t0 * a.dv, live);
            svec = a.vec[nc * 128 + (threadIdx.x & 127)];
        }
    };
    // What a lane adds to a tile's start.
    const int k_row = Rows::row_base(lr, g), k_col = Rows::column_base(lr, g), s_col = Square::column_base(lr, g);
    const int o_at = Square::block_base(16 * wave, lr, g);
    if (from < chunks)
        for (int p = 0; p < 4; ++p) fetch(chunks - 1, p);
    for (int c = chunks - 1; c >= from; --c) {
        unsigned char* buf = lds + (L::kBuffers == 2 ? (c & 1) * L::kBytes : 0);
        if (L::kBuffers == 1 && c < chunks - 1) __syncthreads();  // the chunk before is done with the buffer
        sk.put(buf + L::kK);
        sq.put(buf + L::kQ);
        stm.put(buf + L::kT);
        smm.put(buf + L::kM);
        so.put(buf + L::kV);
        reinterpret_cast<float*>(buf + L::kVec)[threadIdx.x & 127] = svec;
        const int next = c > from ? c - 1 : c;  // the last chunk's loads are not used
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
        Three s[NS];
        float* ds = w.ds + (nc * a.dvp + col) * DK + 8 * g;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            operand(dS[2 * i], dS[2 * i + 1], odd, s[i]);
            if constexpr (!kMaps) store_run(ds + 32 * i, dS[2 * i], dS[2 * i + 1], odd, s[i]);
        }
        stage_wall();
        fetch(next, 0);
        Three mf[4], mg[2];
        f32x4 zb[4];
        auto scores = [&] {
#pragma unroll
            for (int b = 0; b < 4; ++b) mf[b] = Square::template transposed_parts<3>(buf + L::kM, s_col, 1, b);
#pragma unroll
            for (int b = 0; b < 2; ++b) mg[b] = Square::template transposed_parts<3>(buf + L::kM, s_col, 0, b);
        };
        if (!kLate) scores();
#pragma unroll
        for (int b = 0; b < 4; ++b) zb[b] = *reinterpret_cast<const f32x4*>(E + 64 + tok(b, 4 * g));
        // dO as it is, and as E dO scale.
        One od[2];
        Three eo[2];
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
        if (kLate) scores();
        stage_wall();
        fetch(next, 1);
        Three tf[4], tg[2];
        auto inverse = [&] {
#pragma unroll
            for (int b = 0; b < 4; ++b) tf[b] = Square::template transposed_parts<3>(buf + L::kT, s_col, 1, b);
#pragma unroll
            for (int b = 0; b < 2; ++b) tg[b] = Square::template transposed_parts<3>(buf + L::kT, s_col, 0, b);
        };
        if (!kLate) inverse();
#pragma unroll
        for (int b = 0; b < 4; ++b) x[b] = mac(mf[b], od[1], x[b] * zb[b]);
#pragma unroll
        for (int b = 0; b < 2; ++b) x[b] = mac(mg[b], od[0], x[b]);
        if (kLate) inverse();
        Three y[2];
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) operand(x[2 * kk], x[2 * kk + 1], odd, y[kk]);
        stage_wall();
        fetch(next, 2);
        One qc[2][DK / 16];
        auto queries = [&] {
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int i = 0; i < DK / 16; ++i) qc[kk][i] = Rows::transposed(buf + L::kQ, k_col, kk, i);
        };
        if (!kLate) queries();
        // dD = T^T dY.
#pragma unroll
        for (int b = 0; b < 4; ++b) x[b] = mac(tf[b], y[1], zero);
#pragma unroll
        for (int b = 0; b < 2; ++b) x[b] = mac(tg[b], y[0], x[b]);
        if (kLate) queries();
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
        Three d[2];
        float* dd = w.dd + (nc * a.dvp + col) * kChunk + 8 * g;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            if constexpr (!kMaps) {
                OneT<float> run;
                operand(x[2 * kk], x[2 * kk + 1], odd, run);
                store_run(dd + 32 * kk, run);
            }
            operand(x[2 * kk] * -e[2 * kk], x[2 * kk + 1] * -e[2 * kk + 1], odd, d[kk]);
        }
        stage_wall();
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
            for (int i = 0; i < DK / 16; ++i) dS[i] = mac(kc[kk][i], d[kk], dS[i]);
    }
    if (!kMaps && seg == 0 && cb == 0) {
        // Chunks past the stream's last have no gradients; nor have those of a key stream past all of its.
        const int64_t end = int64_t(all) * kChunk, i0 = threadIdx.x;
        if (w.dv)
            for (int64_t i = end * a.dv + i0; i < a.T * a.dv; i += kThreads)
                store_val(static_cast<TIn*>(w.dv) + n * a.T * a.dv + i, 0.f);
        for (void* p : {w.dgate, w.dbeta})
            for (int64_t t = end + i0; p && t < a.T; t += kThreads) store_gate(p, n * a.T + t, a.gate_f32, 0.f);
        if (n % a.group == 0) {
            int64_t most = 0;
            for (int h = 0; h < a.group; ++h) {
                const int64_t l = a.len_of(n + h);
                most = l > most ? l : most;
            }
            for (void* p : {w.dq, w.dk})
                for (int64_t i = (most + kChunk - 1) / kChunk * kChunk * a.dk + i0; p && i < a.T * a.dk; i += kThreads)
                    store_val(static_cast<TIn*>(p) + nk * a.T * a.dk + i, 0.f);
        }
    }
    float* to = kMaps ? a.map_x + (n * a.segs + seg) * a.dk * a.dv : seg == 0 ? w.dstate : nullptr;
    if (!to || !active || col >= a.dv) return;
    if (!kMaps) to += n * a.dk * a.dv;
#pragma unroll
    for (int i = 0; i < DK / 16; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = tok(i, 4 * g + r);
            if (row < a.dk) to[row * a.dv + col] = dS[i][r];
        }
}

// ---- the chunks' gradients ----

// Workgroups that stay, one a CU of an MI355X, each taking every 256th chunk: the
// next slice's rows are on their way while a slice is worked on.  (A workgroup a
// chunk, one resident a CU for its LDS, waited for its loads two thirds of its time: with
// rows kept in bf16, 8 x 16 streams of 4096 tokens 700 us for 669.)
constexpr int kGradWorkgroups = 256;

// Columns of the state a step takes, for the LDS, and threads (1024 have 128 registers
// each: the rows on their way spill).
constexpr int kSlice = 32;
constexpr int kGradThreads = 512;

// P: parts of computed values.
template <typename TIn, int DK, int P>
struct GradLds {
    static constexpr int SL = kSlice, kS = int(sizeof(TIn)), kP = sizeof(TIn) == 2 ? P : 1;  // planes
    using Out = Tile<TIn, sizeof(TIn) == 2 ? 64 : SL>;  // rows of a slice of dO
    static constexpr int kStPlane = SL * DK * kS, kYtPlane = SL * kChunk * kS, kSquare = kPartsBytes<TIn, 64, P>;
    static constexpr int kK = 0, kQ = Tile<TIn, DK>::kBytes, kSt = 2 * kQ, kDs = kSt + kP * kStPlane;
    static constexpr int kYt = kDs + kP * kStPlane, kDd = kYt + kP * kYtPlane, kO = kDd + kP * kYtPlane, kEnd = kO + Out::kBytes;
    static constexpr int kSumBytes = int(sizeof(double)) * kChunk + int(sizeof(float)) * (21 * kChunk + 16);
    // L and X, over the slices' tiles where there is no more LDS: a barrier more.
    static constexpr bool kOver = kEnd + 2 * kSquare + kSumBytes > kGfx950LdsBytes;
    static constexpr int kL = kOver ? kSt : kEnd, kX = kL + kSquare, kSums = kOver ? kEnd : kX + kSquare;
    static constexpr int kBytes = kSums + kSumBytes;
    static_assert(!kOver || kX + kSquare <= kO);
};

// Dense rows of K fp32 values in memory, ROWS of them, to a tile in P planes, PLANE bytes apart.
template <typename E, int K, int ROWS, int NT, int P, int PLANE = Tile<E, K>::kBytes>
struct StageDense {
    static constexpr int kTotal = ROWS * K / 4, kPer = (kTotal + NT - 1) / NT;
    f32x4 x[kPer];
    // `rows` of them, zeros behind.
    __device__ __forceinline__ void load(const float* p, int rows, int tid) {
        const auto r = mfma::make_rsrc(p, rows * K * 4);
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (kTotal % NT == 0 || tid + i * NT < kTotal)
                x[i] = __builtin_bit_cast(f32x4, mfma::buf_load16<mfma::kPolicyDefault>(r, 16 * (tid + i * NT)));
    }
    __device__ __forceinline__ void put(unsigned char* t, int tid) const {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int q = tid + i * NT;
            if (kTotal % NT == 0 || q < kTotal)
                Tile<E, K>::template put4_parts<P, PLANE>(t, Tile<E, K>::four_at(q / (K / 4), 4 * (q % (K / 4))), x[i]);
        }
    }
};

// 64 rows of `width` values by stride, of which `live` are there, in K columns; to a tile T.
template <typename TIn, int K, int NT, bool kVec, typename T = Tile<TIn, K>>
struct RowPieces {
    static constexpr int kVecs = Eight<TIn>::kVecs, kTotal = kChunk * (K / 8), kPer = (kTotal + NT - 1) / NT;
    std::conditional_t<kVec, Eight<TIn>, Ragged<TIn>> x[kPer];
    int stride_, width_, at_;  // of the rows loaded
    __device__ __forceinline__ void load(const TIn* p, int64_t stride, int live, int width, int tid) {
        stride_ = int(stride), width_ = width, at_ = 0;
        __amdgpu_buffer_rsrc_t r;
        if constexpr (kVec)
            r = mfma::make_rsrc(p, ((live - 1) * stride + width) * int(sizeof(TIn)));
        else
            r = ragged_view(p, stride, live, width, at_);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int q = tid + i * NT, row = q / (K / 8), u = q % (K / 8);
            if (kTotal % NT != 0 && q >= kTotal) continue;
            if constexpr (kVec) {
#pragma unroll
                for (int j = 0; j < kVecs; ++j)
                    x[i].v[j] = mfma::buf_load16<mfma::kPolicyDefault>(r, piece_at<TIn>(row, stride_, 8 * u + 4 * j, width));
            } else {
                x[i].load(r, at_ + row * stride_, 8 * u, width, row < live);
            }
        }
    }
    __device__ __forceinline__ void put(unsigned char* t, int tid) const {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int q = tid + i * NT, row = q / (K / 8), u = q % (K / 8);
            if (kTotal % NT != 0 && q >= kTotal) continue;
            Eight<TIn> e;
            if constexpr (kVec)
                e = x[i];
            else
                e = x[i].get(at_ + row * stride_, 8 * u, width_);
#pragma unroll
            for (int j = 0; j < kVecs; ++j) *reinterpret_cast<uint4*>(t + T::at(row, kVecs * u + j)) = e.v[j];
        }
    }
};

// What a workgroup does between two barriers: a slice of the value columns of a
// stream in a chunk.  Only live ones are taken: the walk wrote the zeros of the rest.
struct GradUnit {
    int item, nk, c, h, v0, live;  // item: key stream and chunk
};
__device__ __forceinline__ int live_rows(const DeltaArgs& a, int nk, int c, int h) {
    const int64_t l = a.len_of(int64_t(nk) * a.group + h) - int64_t(c) * kChunk;
    return l < 0 ? 0 : l < kChunk ? int(l) : kChunk;
}
// The next live stream of the unit's chunk or, past its last, of a chunk to come.
__device__ __forceinline__ bool next_stream(const DeltaArgs& a, int items, GradUnit& u) {
    u.v0 = 0;
    while (true) {
        if (++u.h >= a.group) {
            u.h = 0;
            u.item += gridDim.x;
            if (u.item >= items) return false;
            u.nk = unsigned(u.item) / unsigned(a.chunks), u.c = u.item - u.nk * a.chunks;
        }
        u.live = live_rows(a, u.nk, u.c, u.h);
        if (u.live > 0) return true;
    }
}

// Wave (th, dq): TB blocks of 16 tokens and a quarter of the key columns; of the 64 x
// 64 matrices its tokens' rows and 16 columns.  kShared: key streams with several
// value streams, whose dQ and dK are summed in registers.
template <typename TIn, int DK, int kParts, bool kVec, bool kVecV, bool kShared>
__global__ __launch_bounds__(kGradThreads) void delta_grads_kernel(const DeltaBwdArgs w, int items) {
    extern __shared__ __align__(16) unsigned char lds[];
    const DeltaArgs& a = w.f;
    using L = GradLds<TIn, DK, kParts>;
    using Rows = Tile<TIn, DK>;
    using Square = Tile<TIn, 64>;
    using Out = typename L::Out;
    using One = OneT<TIn>;
    using Many = PartsT<TIn, kParts>;
    constexpr int NB = DK / 64, SL = L::SL, NT = kGradThreads, NW = NT / 64, TB = 16 / NW;
    double* G = reinterpret_cast<double*>(lds + L::kSums);
    float* beta = reinterpret_cast<float*>(G + kChunk);
    float* row_sum = beta + kChunk;         // [4][64]
    float* col_sum = row_sum + 4 * kChunk;  // [4 / TB][64]
    float* b_sum = col_sum + 4 * kChunk;    // [4 / TB][64]
    float* dots = b_sum + 4 * kChunk;       // [2][4][64]
    float* ss = dots + 8 * kChunk;          // [NW]
    int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), th = wave >> 2, dq = wave & 3;
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};

    StageDense<TIn, DK, SL, NT, kParts, L::kStPlane> ps, pd;
    StageDense<TIn, 64, SL, NT, kParts, L::kYtPlane> py, pdd;
    RowPieces<TIn, SL, NT, kVecV, Out> po;
    RowPieces<TIn, DK, NT, kVec> pk, pq;
    uint32_t pg = 0, pb = 0;
    // The loads of a unit: its slice, with a stream's first the gates, with a chunk's first K and Q.
    auto prefetch = [&](const GradUnit& u, bool new_item) {
        const int lane = tid & 63;
        const int64_t nk = u.nk, n = nk * a.group + u.h;
        const int rows = min(SL, a.dvp - u.v0);
        const int64_t t0 = int64_t(u.c) * kChunk, slice = (n * a.chunks + u.c) * a.dvp + u.v0;
        if (new_item) {
            int most = u.live;  // of the chunk's first live stream, and of those after it
            for (int h = u.h + 1; a.live.lengths && h < a.group; ++h) most = max(most, live_rows(a, u.nk, u.c, h));
            pk.load(static_cast<const TIn*>(a.k) + nk * a.kn + t0 * a.kt, a.kt, most, a.dk, tid);
            pq.load(static_cast<const TIn*>(a.q) + nk * a.qn + t0 * a.qt, a.qt, most, a.dk, tid);
        }
        if (u.v0 == 0 && wave == 0) {
            const int64_t at = n * a.T + t0 + lane;
            pg = pb = 0;
            if (lane < u.live) {
                if (a.gate) pg = gate_bits(a.gate, at, a.gate_f32);
                pb = gate_bits(a.beta, at, a.gate_f32);
            }
        }
        ps.load(a.st + slice * DK, rows, tid);
        pd.load(w.ds + slice * DK, rows, tid);
        py.load(a.yt + slice * kChunk, rows, tid);
        pdd.load(w.dd + slice * kChunk, rows, tid);
        po.load(static_cast<const TIn*>(w.dout) + (n * a.T + t0) * a.dv + u.v0, a.dv, u.live, a.dv - u.v0, tid);
    };

    GradUnit u = {int(blockIdx.x) - int(gridDim.x), 0, 0, a.group, 0, 0};
    if (!next_stream(a, items, u)) return;
    bool new_item = true, more = true;
    prefetch(u, true);
    f32x4 gq[TB][NB], gk[TB][NB];
    f32x4 P[TB], H[TB], qs[TB][NB], fs[TB][NB], zs[TB][NB];
    float s_ds = 0.f, gate = 0.f;
    while (more) {
        // A new value each time round, as far as the compiler knows: it would keep every address made of it.
        asm volatile("" : "+v"(tid));
        const int lane = tid & 63, g = lane >> 4, lr = lane & 15;
        const int k_col = Rows::column_base(lr, g), s_col = Square::column_base(lr, g), o_row = Out::row_base(lr, g);
        const int k_row = Rows::row_base(lr, g), s_row = Square::row_base(lr, g);
        const bool first = u.v0 == 0;
        const int64_t nk = u.nk, n = nk * a.group + u.h, t0 = int64_t(u.c) * kChunk;
        const int live = u.live, here = int(a.T - t0 < kChunk ? a.T - t0 : kChunk), v0 = u.v0;
        __syncthreads();  // the unit before is done with the LDS
        if (new_item) {
            pk.put(lds + L::kK, tid);
            pq.put(lds + L::kQ, tid);
#pragma unroll
            for (int i = 0; i < TB; ++i)
#pragma unroll
                for (int b = 0; b < NB; ++b) gq[i][b] = gk[i][b] = zero;
        }
        if (first) {
            if (wave == 0) {
                gate = gate_of(pg, a.gate_f32);
                const double s = lane < live && a.gate ? double(log_decay(gate, a.form)) * kLog2e : 0.0;
                G[lane] = wave_scan(s);
                beta[lane] = gate_of(pb, a.gate_f32);
            }
            s_ds = 0.f;
#pragma unroll
            for (int i = 0; i < TB; ++i) {
                P[i] = H[i] = zero;
#pragma unroll
                for (int b = 0; b < NB; ++b) qs[i][b] = fs[i][b] = zs[i][b] = zero;
            }
        }
#pragma unroll
        for (int i = 0; i < ps.kPer; ++i)
            if (ps.kTotal % NT == 0 || tid + i * NT < ps.kTotal)
#pragma unroll
                for (int r = 0; r < 4; ++r) s_ds = fmaf(ps.x[i][r], pd.x[i][r], s_ds);
        ps.put(lds + L::kSt, tid);
        pd.put(lds + L::kDs, tid);
        py.put(lds + L::kYt, tid);
        pdd.put(lds + L::kDd, tid);
        po.put(lds + L::kO, tid);
        GradUnit next = u;
        next.v0 += SL;
        const bool last = next.v0 >= a.dv;
        more = !last || next_stream(a, items, next);
        new_item = more && next.item != u.item;
        const bool item_done = !more || new_item;
        if (more) prefetch(next, new_item);
        u = next;
        __syncthreads();
        TIn* dv = w.dv ? static_cast<TIn*>(w.dv) + (n * a.T + t0) * a.dv : nullptr;
#pragma unroll
        for (int kk = 0; kk < SL / 32; ++kk) {
            const Many yc = Square::template transposed_parts<kParts, L::kYtPlane>(lds + L::kYt, s_col, kk, dq);
            Many ya[TB], da[TB];
            One oa[TB];
#pragma unroll
            for (int i = 0; i < TB; ++i) {
                const int b = TB * th + i;
                ya[i] = Square::template transposed_parts<kParts, L::kYtPlane>(lds + L::kYt, s_col, kk, b);
                da[i] = Square::template transposed_parts<kParts, L::kYtPlane>(lds + L::kDd, s_col, kk, b);
                oa[i] = Out::one(lds + L::kO, o_row, b, kk);
                P[i] = mac(oa[i], yc, P[i]);
                H[i] = mac(da[i], yc, H[i]);
                // A token's dV: four waves hold the same rows, each writes every fourth run.
                if (dv && ((v0 >> 5) + kk) % 4 == dq && tok(b, lr) < here) {
                    const int cv = v0 + 32 * kk + 8 * g;
                    TIn* o = dv + int64_t(tok(b, lr)) * a.dv + cv;
                    if (kVecV && cv + 8 <= a.dv) {
                        store_run(o, delta::first<1>(da[i]));
                    } else {
                        const auto run = __builtin_bit_cast(Eight<TIn>, delta::first<1>(da[i]));
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
                const Many st = Rows::template transposed_parts<kParts, L::kStPlane>(lds + L::kSt, k_col, kk, dq * NB + b);
                const Many ds = Rows::template transposed_parts<kParts, L::kStPlane>(lds + L::kDs, k_col, kk, dq * NB + b);
#pragma unroll
                for (int i = 0; i < TB; ++i) {
                    qs[i][b] = mac(st, oa[i], qs[i][b]);
                    fs[i][b] = mac(st, da[i], fs[i][b]);
                    zs[i][b] = mac(ds, ya[i], zs[i][b]);
                }
            }
        }
        if (!last) continue;
        if constexpr (L::kOver) __syncthreads();  // the slice's products are done with its tiles
        // Rows tok(TB th + i, 4 g + r), column tok(dq, lr) of the 64 x 64 matrices.
        const int jc = tok(dq, lr);
        {
            const float bj = beta[jc];
            const double Gj = G[jc];
            float in_col = 0.f, in_b = 0.f;
#pragma unroll
            for (int i = 0; i < TB; ++i) {
                f32x4 qk = zero, kk = zero, Lm, Xm;
#pragma unroll
                for (int s = 0; s < DK / 32; ++s) {
                    const One kj = Rows::one(lds + L::kK, k_row, dq, s);
                    qk = mac(Rows::one(lds + L::kQ, k_row, TB * th + i, s), kj, qk);
                    kk = mac(Rows::one(lds + L::kK, k_row, TB * th + i, s), kj, kk);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = tok(TB * th + i, 4 * g + r);
                    const float e = row >= jc ? __builtin_amdgcn_exp2f(float(G[row] - Gj)) : 0.f;
                    const float p = a.scale * e * P[i][r], hm = row > jc ? -e * H[i][r] : 0.f;
                    Lm[r] = bj * p;
                    Xm[r] = bj * hm;
                    // A key stream may go on past this value stream, with any values.
                    const float pair = row >= jc && row < live ? fmaf(p, qk[r], hm * kk[r]) : 0.f;
                    in_b += pair;
                    in_col += bj * pair;
                    const float in_row = row_scan(bj * pair);
                    if (lr == 15) row_sum[dq * kChunk + row] = in_row;
                }
                const int at = Square::four_at(jc, tok(TB * th + i, 4 * g));
                Square::template put4_parts<kParts>(lds + L::kL, at, Lm);
                Square::template put4_parts<kParts>(lds + L::kX, at, Xm);
            }
            in_col += __shfl_xor(in_col, 16);
            in_col += __shfl_xor(in_col, 32);
            in_b += __shfl_xor(in_b, 16);
            in_b += __shfl_xor(in_b, 32);
            if (g == 0) col_sum[th * kChunk + jc] = in_col, b_sum[th * kChunk + jc] = in_b;
        }
        s_ds = wave_sum(s_ds);
        if (lane == 0) ss[wave] = s_ds;
        // What comes from the states, by rows: a token a lane, its key columns in registers.
        const double end = G[63];
#pragma unroll
        for (int i = 0; i < TB; ++i) {
            const int row = tok(TB * th + i, lr);
            const float e = __builtin_amdgcn_exp2f(float(G[row])), z = __builtin_amdgcn_exp2f(float(end - G[row]));
            const float b_row = beta[row];
            float from_s = 0.f, from_z = 0.f;  // of E q.(S dO) - E k.(S dD), and of Z k.(dS' Y)
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int at = Rows::four_at(row, tok(dq * NB + b, 4 * g));
                const f32x4 q4 = Rows::four(lds + L::kQ, at), k4 = Rows::four(lds + L::kK, at);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float qv = qs[i][b][r] * (e * a.scale), fv = fs[i][b][r] * e, zv = zs[i][b][r] * z;
                    from_s = fmaf(q4[r], qv, fmaf(-k4[r], fv, from_s));
                    from_z = fmaf(k4[r], zv, from_z);
                    if constexpr (kShared) {
                        gq[i][b][r] += qv;
                        gk[i][b][r] += fmaf(b_row, zv, -fv);
                    } else {
                        gq[i][b][r] = qv;
                        gk[i][b][r] = fmaf(b_row, zv, -fv);
                    }
                }
            }
            from_s += __shfl_xor(from_s, 16);
            from_s += __shfl_xor(from_s, 32);
            from_z += __shfl_xor(from_z, 16);
            from_z += __shfl_xor(from_z, 32);
            if (g == 0) dots[dq * kChunk + row] = from_s, dots[(4 + dq) * kChunk + row] = from_z;
        }
        __syncthreads();
        if (wave == 0 && (w.dgate || w.dbeta)) {
            const int64_t at = n * a.T + t0 + lane;
            float z = 0.f, cols = 0.f, bs = 0.f;
            double dg = 0.0;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                z += dots[(4 + x) * kChunk + lane];
                dg += double(row_sum[x * kChunk + lane]) + dots[x * kChunk + lane];
            }
#pragma unroll
            for (int x = 0; x < 4 / TB; ++x) cols += col_sum[x * kChunk + lane], bs += b_sum[x * kChunk + lane];
            if (lane >= live) z = 0.f, dg = 0.0;
            if (w.dbeta && lane < here) store_gate(w.dbeta, at, a.gate_f32, lane < live ? bs + z : 0.f);
            if (w.dgate) {
                const float bz = beta[lane] * z;
                const float behind = wave_sum(bz) + __builtin_amdgcn_exp2f(float(end)) * wave_sum(lane < NW ? ss[lane] : 0.f);
                dg -= double(bz) + cols;
                dg = wave_scan(__shfl(dg, 63 - lane));
                dg = __shfl(dg, 63 - lane) + behind;
                float x = lane < live && log_decay(gate, a.form) > kLowestLog ? float(dg) : 0.f;  // constant below
                if (a.form == RACE_GATE_SIGMOID) x *= 1.f / (1.f + expf(gate));
                if (lane < here) store_gate(w.dgate, at, a.gate_f32, x);
            }
        }
        // dQ += L K, dK += L^T Q + (X + X^T) K; a token a lane as above.
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
            for (int i = 0; i < TB; ++i) {
                const int b = TB * th + i;
                const bool low = kk <= (b >> 1), high = kk >= (b >> 1);
                Many l, lt, x, xt;
                if (low) {
                    l = Square::template transposed_parts<kParts>(lds + L::kL, s_col, kk, b);
                    x = Square::template transposed_parts<kParts>(lds + L::kX, s_col, kk, b);
                }
                if (high) {
                    lt = Square::template parts<kParts>(lds + L::kL, s_row, b, kk);
                    xt = Square::template parts<kParts>(lds + L::kX, s_row, b, kk);
                }
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    const One kf = Rows::transposed(lds + L::kK, k_col, kk, dq * NB + nb);
                    if (low) {
                        gq[i][nb] = mac(kf, l, gq[i][nb]);
                        gk[i][nb] = mac(kf, x, gk[i][nb]);
                    }
                    if (high) {
                        gk[i][nb] = mac(kf, xt, gk[i][nb]);
                        gk[i][nb] = mac(Rows::transposed(lds + L::kQ, k_col, kk, dq * NB + nb), lt, gk[i][nb]);
                    }
                }
            }
        }
        if (kShared && !item_done) continue;
#pragma unroll
        for (int i = 0; i < TB; ++i) {
            const int row = tok(TB * th + i, lr);
            if (row >= here) continue;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int cd = tok(dq * NB + b, 4 * g), there = a.dk - cd;
                if (there <= 0) continue;
                const int64_t at = (nk * a.T + t0 + row) * a.dk + cd;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    TIn* p = static_cast<TIn*>(x ? w.dk : w.dq);
                    if (!p) continue;
                    const f32x4 v = x ? gk[i][b] : gq[i][b];
                    if (kVec) {
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
}

template <typename TIn, int DK, int P, bool kVec, bool kVecV>
hipError_t launch_grads(const DeltaRule& r, const DeltaBwdArgs& w, hipStream_t stream) {
    constexpr int grads = GradLds<TIn, DK, P>::kBytes;
    static_assert(grads <= kGfx950LdsBytes, "gfx950 gives a workgroup at most 160 KB of LDS");
    const int items = int(r.Nk * w.f.chunks);
    const unsigned grid = unsigned(items < kGradWorkgroups ? items : kGradWorkgroups);
    constexpr bool kAll = kVec && kVecV;  // others have one form
    if (w.f.group > 1 || !kAll)
        delta_grads_kernel<TIn, DK, P, kVec, kVecV, true><<<grid, kGradThreads, grads, stream>>>(w, items);
    else
        delta_grads_kernel<TIn, DK, P, kVec, kVecV, !kAll><<<grid, kGradThreads, grads, stream>>>(w, items);
    return hipGetLastError();
}

template <typename TIn, int DK, bool kVec, bool kVecV>
hipError_t launch_backward(const DeltaRule& r, const DeltaBwdArgs& w, hipStream_t stream) {
    using L = BwdWalkLds<TIn, DK>;
    constexpr int walk = L::kBuffers * L::kBytes;
    static_assert(walk <= kGfx950LdsBytes, "gfx950 gives a workgroup at most 160 KB of LDS");
    auto grid_of = [&](int64_t streams) { return unsigned((streams + 7) / 8 * 8 * ((r.dv + 63) / 64)); };
    if (w.f.segs > 1) {
        delta_bwd_walk_kernel<TIn, DK, kVec, kVecV, true><<<grid_of(r.N * (w.f.segs - 1)), kThreads, walk, stream>>>(w);
        DeltaArgs join = w.f;
        join.state = w.dfinal;
        launch_join<DK, true>(r, join, stream);
    }
    delta_bwd_walk_kernel<TIn, DK, kVec, kVecV, false><<<grid_of(r.N * w.f.segs), kThreads, walk, stream>>>(w);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    if (!w.dq && !w.dk && !w.dv && !w.dgate && !w.dbeta) return hipSuccess;
    // Gradients that are all rounded to bf16 right away take two parts, those of fp32 gates three.
    if constexpr (sizeof(TIn) == 2) {
        if (w.f.gate_f32) return launch_grads<TIn, DK, 3, kVec, kVecV>(r, w, stream);
    }
    return launch_grads<TIn, DK, 2, kVec, kVecV>(r, w, stream);
}

template <typename TIn, bool kVec, bool kVecV>
hipError_t launch_by_width(const DeltaRule& r, const DeltaBwdArgs& w, hipStream_t stream) {
    return r.dk <= 64 ? launch_backward<TIn, 64, kVec, kVecV>(r, w, stream) : launch_backward<TIn, 128, kVec, kVecV>(r, w, stream);
}
template <typename TIn>
hipError_t launch_by_pieces(const DeltaRule& r, const DeltaBwdArgs& w, hipStream_t stream) {
    if (!w.f.vec_k) return launch_by_width<TIn, false, false>(r, w, stream);
    return w.f.vec_o ? launch_by_width<TIn, true, true>(r, w, stream) : launch_by_width<TIn, true, false>(r, w, stream);
}

}  // namespace

int64_t delta_bwd_bytes(const DeltaRule& r) {
    const int64_t nc = r.N * delta_chunks(r), dvp = (r.dv + 15) / 16 * 16;
    const DeltaLayout l = delta_layout(r);
    // With segments, their ends and what they add to a gradient.
    return round256(nc * dvp * dk_padded(r) * 4) + round256(nc * dvp * kChunk * 4) + (l.map_bytes - l.starts);
}

hipError_t launch_delta_bwd(const DeltaRule& r, const DeltaInputs& in, const void* dout, const float* dfinal,
                            const void* records, const DeltaGrads& g, void* scratch, hipStream_t stream) {
    DeltaBwdArgs w = {};
    w.f = delta_args(r, in);
    const DeltaLayout l = delta_layout(r);
    unsigned char* base = const_cast<unsigned char*>(static_cast<const unsigned char*>(records));
    w.f.tm = base, w.f.mm = base + l.mm, w.f.vec = reinterpret_cast<float*>(base + l.vec);
    w.f.st = reinterpret_cast<float*>(base + l.solve_bytes), w.f.yt = reinterpret_cast<float*>(base + l.yt);
    w.dout = dout, w.dfinal = dfinal;
    const int64_t nc = r.N * w.f.chunks;
    w.ds = static_cast<float*>(scratch);
    w.dd = w.ds + round256(nc * w.f.dvp * dk_padded(r) * 4) / 4;
    w.f.segs = l.segs, w.f.seg_chunks = l.seg_chunks;
    if (l.segs > 1) {
        w.f.map_a = reinterpret_cast<float*>(base + l.map_a);
        w.f.starts = w.dd + round256(nc * w.f.dvp * kChunk * 4) / 4;
        w.f.map_x = w.f.starts + (l.map_x - l.starts) / 4;
    }
    w.dq = g.dq, w.dk = g.dk, w.dv = g.dv, w.dgate = g.dgate, w.dbeta = g.dbeta, w.dstate = g.dstate;
    return r.dtype == RACE_BF16 ? launch_by_pieces<bf16_t>(r, w, stream) : launch_by_pieces<float>(r, w, stream);
}

}  // namespace race
