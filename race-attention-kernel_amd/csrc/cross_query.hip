// cross_query.hip -- a few queries of every stream against its kept sums:
//
//     out[t][c] = sum_s w[t][s] B[s][c],   w[t][s] = q[t][s] / (A[s] + eps)
//
// the decode step of a decoder over its encoder's state.  Bound by reading the
// states (S d + S floats a stream) once; one launch.  A workgroup takes a stream
// (or a block of its columns, where there are few streams) and up to TT of its
// queries: their weights go to LDS, then lane groups across the columns take
// rows of B in turn, four rows' loads in flight, and the groups' sums are added
// by shuffles within a wave and through LDS over the waves, in a fixed order.
#include <algorithm>

#include "race_internal.h"

namespace race {
namespace {

template <typename TIn, int V, int TT>
__global__ __launch_bounds__(kThreads) void cross_query_kernel(const TIn* __restrict__ q,
                                                               const float* __restrict__ state,
                                                               TIn* __restrict__ out, int64_t T, int S, int d,
                                                               int cols, int lane_shift) {
    extern __shared__ __align__(16) float lds[];
    float* w = lds;             // [TT][S]
    float* part = lds + TT * S; // [waves][TT][cols]
    constexpr int kWaves = kThreads / 64;
    const int64_t n = blockIdx.y, t0 = int64_t(blockIdx.z) * TT;
    const int cnt = int(min<int64_t>(TT, T - t0));
    const int c0 = blockIdx.x * cols, here = min(cols, d - c0);
    const float* B = state + n * (int64_t(S) * d + S);
    const float* A = B + int64_t(S) * d;
    for (int s = threadIdx.x; s < S; s += kThreads) {
        const float den = A[s] + kEps;
#pragma unroll
        for (int t = 0; t < TT; ++t)
            w[t * S + s] = t < cnt ? to_f32(q[(n * T + t0 + t) * S + s]) / den : 0.f;
    }
    const int lanes = 1 << lane_shift, cl = threadIdx.x & (lanes - 1), rg = threadIdx.x >> lane_shift;
    const int groups = kThreads >> lane_shift;
    const bool mine = cl * V < here;
    const float* bp = B + c0 + (mine ? cl * V : 0);
    float acc[TT][V];
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int j = 0; j < V; ++j) acc[t][j] = 0.f;
    __syncthreads();
    constexpr int kAhead = 4;
    for (int s0 = rg; s0 < S; s0 += kAhead * groups) {
        float b[kAhead][V];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int s = min(s0 + u * groups, S - 1);
            if constexpr (V == 4) {
                const float4 f = *reinterpret_cast<const float4*>(bp + int64_t(s) * d);
                b[u][0] = f.x, b[u][1] = f.y, b[u][2] = f.z, b[u][3] = f.w;
            } else {
                b[u][0] = bp[int64_t(s) * d];
            }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (s0 + u * groups >= S) break;
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                const float x = w[t * S + s0 + u * groups];
#pragma unroll
                for (int j = 0; j < V; ++j) acc[t][j] = fmaf(x, b[u][j], acc[t][j]);
            }
        }
    }
    for (int off = lanes; off < 64; off *= 2) {
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
            for (int j = 0; j < V; ++j) acc[t][j] += __shfl_xor(acc[t][j], off);
    }
    if (mine && (threadIdx.x & 63) < unsigned(lanes)) {
        float* p = part + (threadIdx.x >> 6) * TT * cols + cl * V;
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
            for (int j = 0; j < V; ++j) p[t * cols + j] = acc[t][j];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < cnt * here; e += kThreads) {
        const int t = e / here, c = e - t * here;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) s += part[(i * TT + t) * cols + c];
        store_val(out + (n * T + t0 + t) * d + c0 + c, s);
    }
}

template <typename TIn, int V, int TT>
void launch_query(const void* q, const float* state, void* out, const Problem& p, hipStream_t stream) {
    // Few streams: blocks of 32 columns each; at most 64 lanes across one.
    const int cols = std::min(V * 64, p.N < 256 ? 32 : p.d);
    int lane_shift = 0;
    while ((V << lane_shift) < std::min(cols, p.d)) ++lane_shift;
    const dim3 grid(unsigned((p.d + cols - 1) / cols), unsigned(p.N), unsigned((p.T + TT - 1) / TT));
    const size_t lds = size_t(TT * p.S + kThreads / 64 * TT * cols) * sizeof(float);
    cross_query_kernel<TIn, V, TT><<<grid, kThreads, lds, stream>>>(static_cast<const TIn*>(q), state,
                                                                    static_cast<TIn*>(out), p.T, p.S, p.d, cols,
                                                                    lane_shift);
}

template <typename TIn, int V>
void launch_query_t(const void* q, const float* state, void* out, const Problem& p, hipStream_t stream) {
    if (p.T == 1) return launch_query<TIn, V, 1>(q, state, out, p, stream);
    if (p.T <= 4) return launch_query<TIn, V, 4>(q, state, out, p, stream);
    return launch_query<TIn, V, 16>(q, state, out, p, stream);
}

}  // namespace

hipError_t launch_cross_query(const void* q, const float* state, void* out, const Problem& p, hipStream_t stream) {
    // Rows of B and the states themselves start on 16 bytes.
    const bool four = p.d % 4 == 0 && p.S * (p.d + 1) % 4 == 0;
    if (p.dtype == RACE_BF16)
        four ? launch_query_t<bf16_t, 4>(q, state, out, p, stream) : launch_query_t<bf16_t, 1>(q, state, out, p, stream);
    else
        four ? launch_query_t<float, 4>(q, state, out, p, stream) : launch_query_t<float, 1>(q, state, out, p, stream);
    return hipGetLastError();
}

}  // namespace race
