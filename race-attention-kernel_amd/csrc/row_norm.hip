// row_norm.hip -- norms of whole rows around a recurrent layer, and their gradients.
//
// On the way in (add_norm), over rows of up to 16384 values:
//     s = x + residual        (rounded to the rows' type: the residual stream)
//     y = s r w,              r = 1 / sqrt(mean(s^2) + eps)
// and with y in 8 bits (e4m3), for an 8-bit projection, over a row or a group
// of its columns:
//     scale = max |y| / 448,  y8 = e4m3(y / scale).
// On the way out (gate_norm), over head rows of up to 256 values, from a
// recurrence's streams [B * H][T][d] to rows [B][T][H][d]:
//     y = x r w silu(z),      silu(z) = z / (1 + exp(-z)).
// With u = x r and g the upstream row times w (and silu(z)):
//     dx = r (g - u mean(g u)),   dw = sum over rows of dy u (silu(z)),
//     dz = dy u w sigma (1 + z (1 - sigma)),
// and the gradient of the residual stream itself is added to dx.
//
// Bound by memory: every row is read once and written once.  67 million bf16 values in
// rows of 2048, forward 537 MB in 92 us and backward in 116; in head rows of 128 with
// the gate 403 MB in 93 and 671 MB in 139.  A row of add_norm lies in the registers
// of a wave or of a workgroup, a head row in those of a few lanes; the weights stay in registers while the workgroups walk over rows.
// Sums are fp32 in a fixed order.  The weights' gradients are summed per lane,
// per workgroup through LDS, then over the workgroups by column_sums_kernel.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "row_run.h"

namespace race {
namespace {

template <int V>
__device__ __forceinline__ void load_weight_run(float (&x)[V], const void* w, int w_f32, int64_t c, bool in) {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = in ? 1.f : 0.f;
    if (!w || !in) return;
    if (w_f32) {
        constexpr int kPer = V >= 4 ? 4 : V;
#pragma unroll
        for (int i = 0; i < V; i += kPer) {
            Run<float, kPer> r;
            r.load(static_cast<const float*>(w) + c + i);
#pragma unroll
            for (int j = 0; j < kPer; ++j) x[i + j] = r.get(j);
        }
    } else {
        Run<bf16_t, V> r;
        r.load(static_cast<const bf16_t*>(w) + c);
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = r.get(i);
    }
}

__device__ __forceinline__ float lanes_sum(float x, int shift) {
    for (int k = 0; k < shift; ++k) x += __shfl_xor(x, 1 << k);
    return x;
}
__device__ __forceinline__ uint32_t lanes_max(uint32_t x, int shift) {
    for (int k = 0; k < shift; ++k) x = max(x, uint32_t(__shfl_xor(int(x), 1 << k)));
    return x;
}

// Sums and maxima over the NT threads of a row.  Rows of several waves meet in
// LDS: two arrays taken in turn, so that one barrier a reduction is enough.
template <int NT>
struct RowReduce {
    static constexpr int kWaves = NT / 64;
    uint32_t* lds;  // [2][kWaves][2]
    int parity = 0;
    __device__ __forceinline__ explicit RowReduce(uint32_t* l) : lds(l) {}
    __device__ __forceinline__ void sum2(float& a, float& b) {
        a = lanes_sum(a, 6), b = lanes_sum(b, 6);
        if constexpr (kWaves > 1) {
            uint32_t* at = lds + parity * 2 * kWaves;
            parity ^= 1;
            if ((threadIdx.x & 63) == 0) {
                at[threadIdx.x >> 6] = __float_as_uint(a);
                at[kWaves + (threadIdx.x >> 6)] = __float_as_uint(b);
            }
            __syncthreads();
            a = b = 0.f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) a += __uint_as_float(at[w]), b += __uint_as_float(at[kWaves + w]);
        }
    }
    __device__ __forceinline__ float sum(float a) {
        a = lanes_sum(a, 6);
        if constexpr (kWaves > 1) {
            uint32_t* at = lds + parity * 2 * kWaves;
            parity ^= 1;
            if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = __float_as_uint(a);
            __syncthreads();
            a = 0.f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) a += __uint_as_float(at[w]);
        }
        return a;
    }
    __device__ __forceinline__ uint32_t most(uint32_t a) {
        a = lanes_max(a, 6);
        if constexpr (kWaves > 1) {
            uint32_t* at = lds + parity * 2 * kWaves;
            parity ^= 1;
            if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = a;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kWaves; ++w) a = max(a, at[w]);
        }
        return a;
    }
};

struct AddNormArgs {
    const void *x, *residual, *w;
    void *y, *sum;
    float* scales;
    const void *dy, *dsum;  // backward; x is then what was normed
    void* dx;
    float* partial;  // [gridDim.x][D], nullable
    int64_t rows, xs, rs;
    int D, w_f32, group, groups;  // columns and number of a row's 8-bit groups (group 0: the row)
    float eps;
};

// Threads that share a row, rows of a workgroup.
template <int NT>
constexpr int kRowThreads = NT < 256 ? 256 : NT;

// |y| as a bit pattern: ordered as the values, NaN above all.
__device__ __forceinline__ uint32_t magnitude(float y) { return __float_as_uint(y) & 0x7fffffffu; }

// The factor to 8 bits for a largest magnitude, and the scale it leaves.  Finite
// where the magnitude is subnormal; zero for rows of zeros, whose scale is zero.
// Products of bf16 values often lie half way between two values of 8 bits, and the
// factors' rounding decides: y is (s r) w, r rounded once from a mean that is the sum
// times 1 / D, and the factor 448 times the reciprocal, as elementwise passes over rows have
// them, so that both take the same one wherever the sum of squares is the same.
__device__ __forceinline__ float to_e4m3_factor(float most) { return most > 0.f ? fminf(448.f * (1.f / most), FLT_MAX) : 0.f; }

template <int V>
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float (&y)[V], float f) {
    if constexpr (V >= 4) {
        uint32_t w[V / 4];
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            int x = 0;
            x = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i] * f, y[4 * i + 1] * f, x, false);
            x = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2] * f, y[4 * i + 3] * f, x, true);
            w[i] = uint32_t(x);
        }
        if constexpr (V == 8)
            *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        else
            *reinterpret_cast<uint32_t*>(p) = w[0];
    } else if constexpr (V == 2) {
        *reinterpret_cast<uint16_t*>(p) = uint16_t(__builtin_amdgcn_cvt_pk_fp8_f32(y[0] * f, y[1] * f, 0, false));
    } else {
        *p = uint8_t(__builtin_amdgcn_cvt_pk_fp8_f32(y[0] * f, 0.f, 0, false) & 0xff);
    }
}

// The mean rounded before eps is added, and the root once (rsqrtf is a step off now and then).
__device__ __forceinline__ float mean_and_eps(float sum, float inv_d, float eps) {
#pragma clang fp contract(off)
    const float mean = sum * inv_d;
    return mean + eps;
}
__device__ __forceinline__ float rounded_rsqrt(float x) { return float(rsqrt(double(x))); }

// NP pieces of V values per thread, piece j at column (j NT + thread) V.
template <typename TIn, int V, int NP, int NT, bool kE4m3>
__global__ __launch_bounds__(kRowThreads<NT>) void add_norm_kernel(const AddNormArgs a) {
    using X = Run<TIn, V>;
    __shared__ uint32_t lds[4 * (kRowThreads<NT> / 64)];
    constexpr int kRows = kRowThreads<NT> / NT;
    RowReduce<NT> reduce(lds);
    const int l = threadIdx.x % NT;
    float w[NP][V];
    int c[NP];
    bool in[NP];
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        c[j] = (j * NT + l) * V, in[j] = c[j] < a.D;
        load_weight_run<V>(w[j], a.w, a.w_f32, c[j], in[j]);
    }
    const float inv_d = 1.f / float(a.D);
    for (int64_t row = int64_t(blockIdx.x) * kRows + threadIdx.x / NT; row < a.rows; row += int64_t(gridDim.x) * kRows) {
        const TIn* xp = static_cast<const TIn*>(a.x) + row * a.xs;
        const TIn* rp = static_cast<const TIn*>(a.residual) + row * a.rs;
        float s[NP][V], ss = 0.f;
        X x[NP], res[NP];
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            x[j].clear(), res[j].clear();
            if (in[j]) x[j].load(xp + c[j]);
            if (in[j] && a.residual) res[j].load(rp + c[j]);
        }
#pragma unroll
        for (int j = 0; j < NP; ++j) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                s[j][i] = x[j].get(i);
                if (a.residual) {
                    s[j][i] += res[j].get(i);
                    if constexpr (sizeof(TIn) == 2) s[j][i] = to_f32(f32_to_bf16(s[j][i]));
                }
                ss = fmaf(s[j][i], s[j][i], ss);
            }
            if (a.residual && in[j]) X::store(static_cast<TIn*>(a.sum) + row * a.D + c[j], s[j]);
        }
        const float r = rounded_rsqrt(mean_and_eps(reduce.sum(ss), inv_d, a.eps));
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                s[j][i] = s[j][i] * r * w[j][i];
                if constexpr (kE4m3) most = max(most, in[j] ? magnitude(s[j][i]) : 0u);
            }
            if constexpr (!kE4m3) {
                if (in[j]) X::store(static_cast<TIn*>(a.y) + row * a.D + c[j], s[j]);
            } else if (a.group) {
                // A group is a few consecutive lanes' pieces.
                uint32_t m = 0;
#pragma unroll
                for (int i = 0; i < V; ++i) m = max(m, in[j] ? magnitude(s[j][i]) : 0u);
                const float top = __uint_as_float(lanes_max(m, __builtin_ctz(a.group / V)));
                if (in[j]) {
                    store_e4m3<V>(static_cast<uint8_t*>(a.y) + row * a.D + c[j], s[j], to_e4m3_factor(top));
                    if (c[j] % a.group == 0) a.scales[row * a.groups + c[j] / a.group] = top / 448.f;
                }
            }
        }
        if constexpr (kE4m3) {
            if (!a.group) {
                const float top = __uint_as_float(reduce.most(most)), f = to_e4m3_factor(top);
#pragma unroll
                for (int j = 0; j < NP; ++j)
                    if (in[j]) store_e4m3<V>(static_cast<uint8_t*>(a.y) + row * a.D + c[j], s[j], f);
                if (l == 0) a.scales[row] = top / 448.f;
            }
        }
    }
}

template <typename TIn, int V, int NP, int NT>
__global__ __launch_bounds__(kRowThreads<NT>) void add_norm_bwd_kernel(const AddNormArgs a) {
    using X = Run<TIn, V>;
    __shared__ uint32_t lds[4 * (kRowThreads<NT> / 64)];
    extern __shared__ float rows_dw[];  // [kRows][D], with several rows a workgroup
    constexpr int kRows = kRowThreads<NT> / NT;
    RowReduce<NT> reduce(lds);
    const int l = threadIdx.x % NT;
    float w[NP][V], dw[NP][V];
    int c[NP];
    bool in[NP];
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        c[j] = (j * NT + l) * V, in[j] = c[j] < a.D;
        load_weight_run<V>(w[j], a.w, a.w_f32, c[j], in[j]);
#pragma unroll
        for (int i = 0; i < V; ++i) dw[j][i] = 0.f;
    }
    const float inv_d = 1.f / float(a.D);
    for (int64_t row = int64_t(blockIdx.x) * kRows + threadIdx.x / NT; row < a.rows; row += int64_t(gridDim.x) * kRows) {
        X x[NP], up[NP], ds[NP];
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            x[j].clear(), up[j].clear(), ds[j].clear();
            if (!in[j]) continue;
            x[j].load(static_cast<const TIn*>(a.x) + row * a.xs + c[j]);
            if (a.dy) up[j].load(static_cast<const TIn*>(a.dy) + row * a.D + c[j]);
            if (a.dsum) ds[j].load(static_cast<const TIn*>(a.dsum) + row * a.D + c[j]);
        }
        float ss = 0.f, gx = 0.f;
#pragma unroll
        for (int j = 0; j < NP; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float xv = x[j].get(i);
                ss = fmaf(xv, xv, ss);
                gx = fmaf(up[j].get(i) * w[j][i], xv, gx);
            }
        reduce.sum2(ss, gx);
        // u = x r: dx = r (g w) - x (r^3 sum(g w x) / d).
        const float r = rsqrtf(ss / float(a.D) + a.eps), m = gx * inv_d * r * r * r;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            float dx[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float xv = x[j].get(i), g = up[j].get(i);
                dw[j][i] = fmaf(g, xv * r, dw[j][i]);
                dx[i] = fmaf(g * w[j][i], r, fmaf(-xv, m, ds[j].get(i)));
            }
            if (a.dx && in[j]) X::store(static_cast<TIn*>(a.dx) + row * a.D + c[j], dx);
        }
    }
    if (!a.partial) return;
    float* out = a.partial + int64_t(blockIdx.x) * a.D;
    if constexpr (kRows > 1) {
        float* mine = rows_dw + int(threadIdx.x / NT) * a.D;
#pragma unroll
        for (int j = 0; j < NP; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (in[j]) mine[c[j] + i] = dw[j][i];
        __syncthreads();
        for (int k = threadIdx.x; k < a.D; k += kRowThreads<NT>) {
            float s = 0.f;
#pragma unroll
            for (int q = 0; q < kRows; ++q) s += rows_dw[q * a.D + k];
            out[k] = s;
        }
    } else {
#pragma unroll
        for (int j = 0; j < NP; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (in[j]) out[c[j] + i] = dw[j][i];
    }
}

__global__ __launch_bounds__(1024) void column_sums_kernel(const float* partial, int rows, int d, void* out, int f32) {
    column_sums(partial, rows, d, out, f32);
}

hipError_t launch_column_sums(const float* partial, int rows, int d, void* out, int f32, hipStream_t stream) {
    column_sums_kernel<<<unsigned((d + 31) / 32), 1024, 0, stream>>>(partial, rows, d, out, f32);
    return hipGetLastError();
}

// Whether the rows' pieces of `v` values lie at multiples of their size.
bool add_norm_whole(const AddNorm& n, int v) { return n.D % v == 0 && n.xs % v == 0 && n.rs % v == 0; }
int add_norm_vector(const AddNorm& n) {
    const int wide = n.dtype == RACE_BF16 ? 8 : 4;
    return add_norm_whole(n, wide) ? wide : add_norm_whole(n, 2) ? 2 : 1;
}

// Pieces of 16 bytes where the rows lie so, else of two values or one: 16384 bf16 rows of
// 1000 / 1002 / 1001 values, forward and backward, 47 / 58 / 111 us.
// f(V, NP, NT) as compile-time values for rows of D values in pieces of v: a wave
// a row while it holds the row in 4 pieces a lane, then a workgroup.
template <int V, typename F>
hipError_t by_row(int D, F f) {
    using std::integral_constant;
    const int pieces = (D + V - 1) / V;
    auto call = [&](auto np, auto nt) { return f(integral_constant<int, V>{}, np, nt); };
    constexpr integral_constant<int, 64> wave{};
    constexpr integral_constant<int, 256> four{};
    constexpr integral_constant<int, 1024> all{};
    if (pieces <= 64) return call(integral_constant<int, 1>{}, wave);
    if (pieces <= 128) return call(integral_constant<int, 2>{}, wave);
    if (pieces <= 256) return call(integral_constant<int, 4>{}, wave);
    if (pieces <= 512) return call(integral_constant<int, 2>{}, four);
    if (pieces <= 1024) return call(integral_constant<int, 4>{}, four);
    if constexpr (V == 1) {
        if (pieces > 8192) return call(integral_constant<int, 16>{}, all);
    }
    if constexpr (V <= 2) {
        if (pieces > 4096) return call(integral_constant<int, 8>{}, all);
    }
    if constexpr (V <= 4) {
        if (pieces > 2048) return call(integral_constant<int, 4>{}, all);
    }
    return call(integral_constant<int, 2>{}, all);
}

// Rows of a workgroup of by_row's shape.
int rows_of_workgroup(const AddNorm& n) {
    const int v = add_norm_vector(n);
    return (n.D + v - 1) / v <= 256 ? 4 : 1;
}

// Workgroups that walk over the rows.  Backward, half as many: 9235 rows of 1001 fp32 values
// 34 us against 27; twice as many: 29.  Forward, 1024 .. 4096 are alike (32768 x 2048 bf16: 89 .. 92 us,
// 537 MB; backward 116 us).
constexpr int kAddNormFwdWorkgroups = 2048, kAddNormBwdWorkgroups = 1024;

unsigned add_norm_grid(const AddNorm& n, int most) {
    const int per = rows_of_workgroup(n);
    return unsigned(std::min<int64_t>((n.rows + per - 1) / per, most));
}

AddNormArgs add_norm_args(const AddNorm& n, const void* x, const void* w) {
    AddNormArgs a = {};
    a.x = x, a.w = w;
    a.rows = n.rows, a.xs = n.xs, a.rs = n.rs;
    a.D = n.D, a.w_f32 = n.weight_dtype == RACE_F32, a.group = n.group;
    a.groups = n.group ? (n.D + n.group - 1) / n.group : 1;
    a.eps = n.eps;
    return a;
}

template <typename TIn, typename F>
hipError_t by_piece(const AddNorm& n, F f) {
    constexpr int kWide = sizeof(TIn) == 2 ? 8 : 4;
    const int v = add_norm_vector(n);
    return v == kWide ? by_row<kWide>(n.D, f) : v == 2 ? by_row<2>(n.D, f) : by_row<1>(n.D, f);
}

template <typename TIn>
hipError_t launch_add_norm_t(const AddNorm& n, const AddNormArgs& a, hipStream_t stream) {
    const unsigned grid = add_norm_grid(n, kAddNormFwdWorkgroups);
    return by_piece<TIn>(n, [&](auto v, auto np, auto nt) {
        constexpr int V = decltype(v)::value, NP = decltype(np)::value, NT = decltype(nt)::value;
        if (n.e4m3)
            add_norm_kernel<TIn, V, NP, NT, true><<<grid, kRowThreads<NT>, 0, stream>>>(a);
        else
            add_norm_kernel<TIn, V, NP, NT, false><<<grid, kRowThreads<NT>, 0, stream>>>(a);
        return hipGetLastError();
    });
}

template <typename TIn>
hipError_t launch_add_norm_bwd_t(const AddNorm& n, const AddNormArgs& a, hipStream_t stream) {
    const unsigned grid = add_norm_grid(n, kAddNormBwdWorkgroups);
    return by_piece<TIn>(n, [&](auto v, auto np, auto nt) {
        constexpr int V = decltype(v)::value, NP = decltype(np)::value, NT = decltype(nt)::value;
        constexpr int kRows = kRowThreads<NT> / NT;
        const size_t lds = kRows > 1 && a.partial ? size_t(kRows) * n.D * sizeof(float) : 0;
        add_norm_bwd_kernel<TIn, V, NP, NT><<<grid, kRowThreads<NT>, lds, stream>>>(a);
        return hipGetLastError();
    });
}

// ---- the gated norm of head rows ----

struct GateNormArgs {
    const void *x, *z, *w, *dy;
    void *y, *dx, *dz;
    float* partial;  // [gridDim.x][d], nullable
    int64_t rows;    // B * T * H
    int64_t xn, xt, zb, zt, zh;
    int T, H, d, w_f32, lane_shift;
    float eps;
};

__device__ __forceinline__ float sigmoid_of(float z) {
    const float e = __expf(-fabsf(z));
    const float s = 1.f / (1.f + e);
    return z >= 0.f ? s : e * s;
}

// A lane group a row (NS pieces a lane), in the order of the rows [B][T][H] that
// z and y have.
template <typename TIn, int V, int NS, bool kBack>
__global__ __launch_bounds__(kThreads) void gate_norm_kernel(const GateNormArgs a) {
    using X = Run<TIn, V>;
    extern __shared__ float rows_dw[];  // backward: [lane groups][d]
    const int l = threadIdx.x & ((1 << a.lane_shift) - 1), r0 = threadIdx.x >> a.lane_shift;
    const int per = kThreads >> a.lane_shift;
    float w[NS][V], dw[NS][V];
    int c[NS];
    bool in[NS];
#pragma unroll
    for (int j = 0; j < NS; ++j) {
        c[j] = ((j << a.lane_shift) + l) * V, in[j] = c[j] < a.d;
        load_weight_run<V>(w[j], a.w, a.w_f32, c[j], in[j]);
#pragma unroll
        for (int i = 0; i < V; ++i) dw[j][i] = 0.f;
    }
    const float inv_d = 1.f / float(a.d);
    for (int64_t first = int64_t(blockIdx.x) * per; first < a.rows; first += int64_t(gridDim.x) * per) {
        const int64_t row = first + r0;
        const bool there = row < a.rows;
        int64_t b;
        int t, h;
        if (a.rows < (int64_t(1) << 31)) {  // divisions of 64 bits would cost more than the rest of a short row
            const unsigned bt = unsigned(row) / unsigned(a.H), b32 = bt / unsigned(a.T);
            h = int(unsigned(row) - bt * a.H), t = int(bt - b32 * a.T), b = b32;
        } else {
            const int64_t bt = row / a.H;
            b = bt / a.T;
            h = int(row - bt * a.H), t = int(bt - b * a.T);
        }
        const TIn* xp = static_cast<const TIn*>(a.x) + (b * a.H + h) * a.xn + t * a.xt;
        const TIn* zp = static_cast<const TIn*>(a.z) + b * a.zb + t * a.zt + h * a.zh;
        X x[NS], z[NS], up[NS];
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            x[j].clear(), z[j].clear(), up[j].clear();
            if (!there || !in[j]) continue;
            x[j].load(xp + c[j]), z[j].load(zp + c[j]);
            if constexpr (kBack) up[j].load(static_cast<const TIn*>(a.dy) + row * a.d + c[j]);
        }
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < NS; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) ss = fmaf(x[j].get(i), x[j].get(i), ss);
        const float r = rsqrtf(lanes_sum(ss, a.lane_shift) / float(a.d) + a.eps);
        if constexpr (!kBack) {
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                float y[V];
#pragma unroll
                for (int i = 0; i < V; ++i) y[i] = x[j].get(i) * r * w[j][i] * (z[j].get(i) * sigmoid_of(z[j].get(i)));
                if (there && in[j]) X::store(static_cast<TIn*>(a.y) + row * a.d + c[j], y);
            }
        } else {
            float gx = 0.f, g[NS][V];
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                float dz[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float zv = z[j].get(i), s = sigmoid_of(zv), u = x[j].get(i) * r, o = up[j].get(i);
                    dz[i] = o * u * w[j][i] * (s * fmaf(zv, 1.f - s, 1.f));
                    const float gated = o * (zv * s);
                    dw[j][i] = fmaf(gated, u, dw[j][i]);
                    g[j][i] = gated * w[j][i];
                    gx = fmaf(g[j][i], u, gx);
                }
                if (a.dz && there && in[j]) X::store(static_cast<TIn*>(a.dz) + row * a.d + c[j], dz);
            }
            const float m = lanes_sum(gx, a.lane_shift) * inv_d;
            TIn* dxp = static_cast<TIn*>(a.dx) + ((b * a.H + h) * a.T + t) * a.d;
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                float dx[V];
#pragma unroll
                for (int i = 0; i < V; ++i) dx[i] = r * (g[j][i] - x[j].get(i) * r * m);
                if (a.dx && there && in[j]) X::store(dxp + c[j], dx);
            }
        }
    }
    if constexpr (kBack) {
        if (!a.partial) return;
#pragma unroll
        for (int j = 0; j < NS; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (in[j]) rows_dw[r0 * a.d + c[j] + i] = dw[j][i];
        __syncthreads();
        for (int k = threadIdx.x; k < a.d; k += kThreads) {
            float s = 0.f;
            for (int q = 0; q < per; ++q) s += rows_dw[q * a.d + k];
            a.partial[int64_t(blockIdx.x) * a.d + k] = s;
        }
    }
}

int gate_norm_vector(const GateNorm& n) {
    auto whole = [&](int v) {
        for (int64_t s : {int64_t(n.d), n.xn, n.xt, n.zb, n.zt, n.zh})
            if (s % v != 0) return false;
        return true;
    };
    const int wide = n.dtype == RACE_BF16 ? 8 : 4;
    return whole(wide) ? wide : whole(2) ? 2 : 1;
}

// Lanes of a row: one for each wide piece, or for four narrow ones, so that short rows
// leave a workgroup more of them (262144 rows of 33 bf16 values, forward and backward:
// a piece a lane 75 + 137 us, four 35 + 57).
constexpr int kNarrowPieces = 4;
int lane_shift_of(const GateNorm& n) {
    const int v = gate_norm_vector(n), each = v >= 4 ? 1 : kNarrowPieces, pieces = (n.d + v * each - 1) / (v * each);
    int k = 0;
    while (k < 6 && (1 << k) < pieces) ++k;
    return k;
}

// As add_norm's.  [16 * 12, 577, 96] fp32: forward with 1024 35 us, with 2048 or 4096 28; backward
// with 512, 1024 and 2048 65, 46 and 38.  [8 * 16, 4096, 128] bf16: 92 and 137 us.
constexpr int kGateNormFwdWorkgroups = 2048, kGateNormBwdWorkgroups = 2048;

template <bool kBack>
hipError_t launch_gate_norm_any(const GateNorm& n, GateNormArgs a, int most, unsigned* workgroups, hipStream_t stream) {
    a.rows = n.B * n.T * n.H;
    a.xn = n.xn, a.xt = n.xt, a.zb = n.zb, a.zt = n.zt, a.zh = n.zh;
    a.T = int(n.T), a.H = n.H, a.d = n.d, a.w_f32 = n.weight_dtype == RACE_F32, a.eps = n.eps;
    a.lane_shift = lane_shift_of(n);
    const int per = kThreads >> a.lane_shift;
    const unsigned grid = unsigned(std::min<int64_t>((a.rows + per - 1) / per, most));
    *workgroups = grid;
    const size_t lds = kBack && a.partial ? size_t(per) * n.d * sizeof(float) : 0;
    const int v = gate_norm_vector(n);
    auto launch = [&](auto type, auto pieces, auto per_lane) {
        gate_norm_kernel<decltype(type), decltype(pieces)::value, decltype(per_lane)::value, kBack>
            <<<grid, kThreads, lds, stream>>>(a);
        return hipGetLastError();
    };
    using std::integral_constant;
    auto by_type = [&](auto type) {
        constexpr int kWide = sizeof(type) == 2 ? 8 : 4;
        if (v == kWide) return launch(type, integral_constant<int, kWide>{}, integral_constant<int, 1>{});
        if (v == 2) return launch(type, integral_constant<int, 2>{}, integral_constant<int, kNarrowPieces>{});
        return launch(type, integral_constant<int, 1>{}, integral_constant<int, kNarrowPieces>{});
    };
    return n.dtype == RACE_BF16 ? by_type(bf16_t{}) : by_type(float{});
}

}  // namespace

int64_t add_norm_partial_floats(const AddNorm& n) { return int64_t(add_norm_grid(n, kAddNormBwdWorkgroups)) * n.D; }

hipError_t launch_add_norm(const AddNorm& n, const void* x, const void* residual, const void* w, void* y, float* scales,
                           void* sum, hipStream_t stream) {
    AddNormArgs a = add_norm_args(n, x, w);
    a.residual = residual, a.y = y, a.scales = scales, a.sum = sum;
    return n.dtype == RACE_BF16 ? launch_add_norm_t<bf16_t>(n, a, stream) : launch_add_norm_t<float>(n, a, stream);
}

hipError_t launch_add_norm_bwd(const AddNorm& n, const void* s, const void* w, const void* dy, const void* dsum, void* dx,
                               void* dw, float* partial, hipStream_t stream) {
    AddNormArgs a = add_norm_args(n, s, w);
    a.dy = dy, a.dsum = dsum, a.dx = dx, a.partial = dw ? partial : nullptr;
    const hipError_t err =
        n.dtype == RACE_BF16 ? launch_add_norm_bwd_t<bf16_t>(n, a, stream) : launch_add_norm_bwd_t<float>(n, a, stream);
    if (err != hipSuccess || !dw) return err;
    return launch_column_sums(partial, int(add_norm_grid(n, kAddNormBwdWorkgroups)), n.D, dw, a.w_f32, stream);
}

int64_t gate_norm_partial_floats(const GateNorm& n) { return int64_t(kGateNormBwdWorkgroups) * n.d; }

hipError_t launch_gate_norm(const GateNorm& n, const void* x, const void* z, const void* w, void* y, hipStream_t stream) {
    GateNormArgs a = {};
    a.x = x, a.z = z, a.w = w, a.y = y;
    unsigned grid = 0;
    return launch_gate_norm_any<false>(n, a, kGateNormFwdWorkgroups, &grid, stream);
}

hipError_t launch_gate_norm_bwd(const GateNorm& n, const void* x, const void* z, const void* w, const void* dy, void* dx,
                                void* dz, void* dw, float* partial, hipStream_t stream) {
    GateNormArgs a = {};
    a.x = x, a.z = z, a.w = w, a.dy = dy, a.dx = dx, a.dz = dz, a.partial = dw ? partial : nullptr;
    unsigned grid = 0;
    const hipError_t err = launch_gate_norm_any<true>(n, a, kGateNormBwdWorkgroups, &grid, stream);
    if (err != hipSuccess || !dw) return err;
    return launch_column_sums(partial, int(grid), n.d, dw, n.weight_dtype == RACE_F32, stream);
}

}  // namespace race
