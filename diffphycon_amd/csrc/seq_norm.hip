// Layer norm over the last axis, forward and backward (include/dpc.h: dpc_seq_norm_*).
//   mu = sum x / C, var = sum (x - mu)^2 / C, s = (var + eps)^-1/2, xh = (x - mu) s, y = xh w + b
//   g = dy w, dx = s (g - mean(g) - xh mean(g xh)), dw = sum_rows dy xh, db = sum_rows dy
// Bound by bytes: the forward reads x and writes y, the backward reads x and dy and writes dx, each once.  A row lives in the registers
// of G lanes (4, 16, 64 or a whole workgroup of 256; N accesses of 16 bytes a lane), so that the centred second sum of the variance -- no
// E[x^2] - mu^2 cancellation -- costs no second read.  Rows too wide for that (over 2048 accesses) are read again from L2.
// The backward pass keeps dw and db in registers over all rows of a group, adds the groups of a workgroup in LDS and writes one row of
// partial sums per workgroup; a second kernel adds those in fixed order.
#include <algorithm>

#include "common.h"

namespace dpc {
namespace seqnorm {

template <class T> constexpr int VEC = 16 / (int)sizeof(T);

// Element e of access n of a lane.  Rows that start on 16 bytes and hold whole accesses: 16 consecutive bytes; other rows: one element at a
// time, consecutive lanes on consecutive elements.
template <class T, int G> struct Map {
    int lane; bool vec;
    __device__ __forceinline__ int at(int n, int e) const { return vec ? (n * G + lane) * VEC<T> + e : n * G * VEC<T> + e * G + lane; }
};

template <class T, int G>
__device__ __forceinline__ void load(const T* __restrict__ row, const Map<T, G>& m, int n, int C, float (&v)[VEC<T>]) {
    typedef T Q __attribute__((ext_vector_type(VEC<T>)));
    if (m.vec) {
        const int c = m.at(n, 0);
        if (c < C) {
            const Q q = *reinterpret_cast<const Q*>(row + c);
#pragma unroll
            for (int e = 0; e < VEC<T>; ++e) v[e] = (float)q[e];
            return;
        }
#pragma unroll
        for (int e = 0; e < VEC<T>; ++e) v[e] = 0.f;
    } else {
#pragma unroll
        for (int e = 0; e < VEC<T>; ++e) { const int c = m.at(n, e); v[e] = c < C ? (float)row[c] : 0.f; }
    }
}

template <class T, int G>
__device__ __forceinline__ void store(T* __restrict__ row, const Map<T, G>& m, int n, int C, const float (&v)[VEC<T>]) {
    typedef T Q __attribute__((ext_vector_type(VEC<T>)));
    if (m.vec) {
        const int c = m.at(n, 0);
        if (c < C) {
            Q q;
#pragma unroll
            for (int e = 0; e < VEC<T>; ++e) q[e] = (T)v[e];
            *reinterpret_cast<Q*>(row + c) = q;
        }
    } else {
#pragma unroll
        for (int e = 0; e < VEC<T>; ++e) { const int c = m.at(n, e); if (c < C) row[c] = (T)v[e]; }
    }
}

// weight / bias element, fp32 or T (null: the identity's value)
template <class T> __device__ __forceinline__ float param(const void* w, int w32, int c, float none) {
    return !w ? none : w32 ? reinterpret_cast<const float*>(w)[c] : (float)reinterpret_cast<const T*>(w)[c];
}

template <int G> __device__ __forceinline__ float group_sum(float v, float* s_red) {
#pragma unroll
    for (int x = (G < 64 ? G : 64) / 2; x; x >>= 1) v += __shfl_xor(v, x, 64);
    if (G == 256) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) s_red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = (s_red[0] + s_red[1]) + (s_red[2] + s_red[3]);
    }
    return v;
}

struct FwdParams {
    const void *x, *w, *b;
    void* y;
    float* stats;
    long long rows, xs;
    int C, w32, vec;
    float eps;
};

template <class T, int G, int N>
__global__ __launch_bounds__(256) void fwd_kernel(const FwdParams p) {
    __shared__ float s_red[4];
    constexpr int V = VEC<T>, R = 256 / G;
    const Map<T, G> m{(int)(threadIdx.x & (G - 1)), p.vec != 0};
    const float inv_c = 1.f / (float)p.C;
    for (long long r0 = (long long)blockIdx.x * R; r0 < p.rows; r0 += (long long)gridDim.x * R) {      // (uniform over the workgroup)
        const long long r = r0 + threadIdx.x / G;
        const bool ok = r < p.rows;
        const T* x = reinterpret_cast<const T*>(p.x) + (ok ? r : 0) * p.xs;
        float v[N][V], sum = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            load<T, G>(x, m, n, p.C, v[n]);
#pragma unroll
            for (int e = 0; e < V; ++e) sum += v[n][e];
        }
        const float mu = group_sum<G>(sum, s_red) * inv_c;
        sum = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[n][e] -= mu;
                if (m.at(n, e) < p.C) sum += v[n][e] * v[n][e];
            }
        const float rstd = 1.f / sqrtf(group_sum<G>(sum, s_red) * inv_c + p.eps);
        if (ok) {
            T* y = reinterpret_cast<T*>(p.y) + r * (long long)p.C;
#pragma unroll
            for (int n = 0; n < N; ++n) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const int c = min(m.at(n, e), p.C - 1);
                    v[n][e] = v[n][e] * rstd * param<T>(p.w, p.w32, c, 1.f) + param<T>(p.b, p.w32, c, 0.f);
                }
                store<T, G>(y, m, n, p.C, v[n]);
            }
            if (m.lane == 0) { p.stats[2 * r] = mu; p.stats[2 * r + 1] = rstd; }
        }
    }
}

// rows wider than 2048 accesses: one workgroup a row, three reads of x (the later two from L2)
template <class T>
__global__ __launch_bounds__(256) void fwd_wide_kernel(const FwdParams p) {
    __shared__ float s_red[4];
    constexpr int V = VEC<T>;
    const Map<T, 256> m{(int)threadIdx.x, p.vec != 0};
    const float inv_c = 1.f / (float)p.C;
    const int N = (p.C + 256 * V - 1) / (256 * V);
    for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* x = reinterpret_cast<const T*>(p.x) + r * p.xs;
        float v[V], sum = 0.f;
        for (int n = 0; n < N; ++n) {
            load<T, 256>(x, m, n, p.C, v);
#pragma unroll
            for (int e = 0; e < V; ++e) sum += v[e];
        }
        const float mu = group_sum<256>(sum, s_red) * inv_c;
        sum = 0.f;
        for (int n = 0; n < N; ++n) {
            load<T, 256>(x, m, n, p.C, v);
#pragma unroll
            for (int e = 0; e < V; ++e) if (m.at(n, e) < p.C) sum += (v[e] - mu) * (v[e] - mu);
        }
        const float rstd = 1.f / sqrtf(group_sum<256>(sum, s_red) * inv_c + p.eps);
        T* y = reinterpret_cast<T*>(p.y) + r * (long long)p.C;
        for (int n = 0; n < N; ++n) {
            load<T, 256>(x, m, n, p.C, v);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int c = min(m.at(n, e), p.C - 1);
                v[e] = (v[e] - mu) * rstd * param<T>(p.w, p.w32, c, 1.f) + param<T>(p.b, p.w32, c, 0.f);
            }
            store<T, 256>(y, m, n, p.C, v);
        }
        if (threadIdx.x == 0) { p.stats[2 * r] = mu; p.stats[2 * r + 1] = rstd; }
    }
}

struct BwdParams {
    const void *dy, *x, *w;
    const float* stats;
    void* dx;
    float* part;               // [gridDim.x][2][C] sums of dy xh and dy, or null
    long long rows, dys, xs;
    int C, w32, vec;
};

template <class T, int G, int N>
__global__ __launch_bounds__(256) void bwd_kernel(const BwdParams p) {
    constexpr int V = VEC<T>, R = 256 / G;
    __shared__ float s_red[4];
    __shared__ float s_sum[G < 256 ? 2 * 256 * N * V : 1];
    const Map<T, G> m{(int)(threadIdx.x & (G - 1)), p.vec != 0};
    const float inv_c = 1.f / (float)p.C;
    float dw[N][V], db[N][V];
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int e = 0; e < V; ++e) dw[n][e] = db[n][e] = 0.f;
    for (long long r0 = (long long)blockIdx.x * R; r0 < p.rows; r0 += (long long)gridDim.x * R) {
        const long long r = r0 + threadIdx.x / G;
        const bool ok = r < p.rows;
        const long long at = ok ? r : 0;
        const T* x = reinterpret_cast<const T*>(p.x) + at * p.xs;
        const T* dy = reinterpret_cast<const T*>(p.dy) + at * p.dys;
        const float mu = p.stats[2 * at], rstd = p.stats[2 * at + 1];
        float xh[N][V], g[N][V], a = 0.f, b = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            load<T, G>(x, m, n, p.C, xh[n]);
            load<T, G>(dy, m, n, p.C, g[n]);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int c = m.at(n, e);
                xh[n][e] = (xh[n][e] - mu) * rstd;
                if (c >= p.C) xh[n][e] = 0.f;
                if (ok) { dw[n][e] += g[n][e] * xh[n][e]; db[n][e] += g[n][e]; }
                g[n][e] *= param<T>(p.w, p.w32, min(c, p.C - 1), 1.f);
                a += g[n][e];
                b += g[n][e] * xh[n][e];
            }
        }
        a = group_sum<G>(a, s_red) * inv_c;
        b = group_sum<G>(b, s_red) * inv_c;
        if (ok) {
            T* dx = reinterpret_cast<T*>(p.dx) + r * (long long)p.C;
#pragma unroll
            for (int n = 0; n < N; ++n) {
#pragma unroll
                for (int e = 0; e < V; ++e) xh[n][e] = rstd * (g[n][e] - a - xh[n][e] * b);
                store<T, G>(dx, m, n, p.C, xh[n]);
            }
        }
    }
    if (!p.part) return;
    float* part = p.part + (long long)blockIdx.x * 2 * p.C;
    if (G == 256) {
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int c = m.at(n, e);
                if (c < p.C) { part[c] = dw[n][e]; part[p.C + c] = db[n][e]; }
            }
        return;
    }
    constexpr int W = G * N * V;                                     // columns a group holds
    const int grp = threadIdx.x / G;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            s_sum[(grp * N * V + n * V + e) * G + m.lane] = dw[n][e];
            s_sum[((R + grp) * N * V + n * V + e) * G + m.lane] = db[n][e];
        }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * W; i += 256) {
        const int half = i / W, k = i % W;                           // k = (n * V + e) * G + lane
        float sum = 0.f;
#pragma unroll
        for (int q = 0; q < R; ++q) sum += s_sum[(half * R + q) * W + k];
        const Map<T, G> mm{k % G, p.vec != 0};
        const int c = mm.at(k / G / V, k / G % V);
        if (c < p.C) part[half * p.C + c] = sum;
    }
}

template <class T>
__global__ __launch_bounds__(256) void bwd_wide_kernel(const BwdParams p) {
    __shared__ float s_red[4];
    constexpr int V = VEC<T>;
    const Map<T, 256> m{(int)threadIdx.x, p.vec != 0};
    const float inv_c = 1.f / (float)p.C;
    const int N = (p.C + 256 * V - 1) / (256 * V);
    float* part = p.part ? p.part + (long long)blockIdx.x * 2 * p.C : nullptr;
    bool first = true;
    for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* x = reinterpret_cast<const T*>(p.x) + r * p.xs;
        const T* dy = reinterpret_cast<const T*>(p.dy) + r * p.dys;
        const float mu = p.stats[2 * r], rstd = p.stats[2 * r + 1];
        float xh[V], g[V], a = 0.f, b = 0.f;
        for (int n = 0; n < N; ++n) {
            load<T, 256>(x, m, n, p.C, xh);
            load<T, 256>(dy, m, n, p.C, g);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int c = m.at(n, e);
                if (c >= p.C) continue;
                xh[e] = (xh[e] - mu) * rstd;
                if (part) {                                          // (this thread's own columns: no other touches them)
                    part[c] = (first ? 0.f : part[c]) + g[e] * xh[e];
                    part[p.C + c] = (first ? 0.f : part[p.C + c]) + g[e];
                }
                g[e] *= param<T>(p.w, p.w32, c, 1.f);
                a += g[e];
                b += g[e] * xh[e];
            }
        }
        first = false;
        a = group_sum<256>(a, s_red) * inv_c;
        b = group_sum<256>(b, s_red) * inv_c;
        T* dx = reinterpret_cast<T*>(p.dx) + r * (long long)p.C;
        for (int n = 0; n < N; ++n) {
            load<T, 256>(x, m, n, p.C, xh);
            load<T, 256>(dy, m, n, p.C, g);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int c = min(m.at(n, e), p.C - 1);
                xh[e] = rstd * (g[e] * param<T>(p.w, p.w32, c, 1.f) - a - (xh[e] - mu) * rstd * b);
            }
            store<T, 256>(dx, m, n, p.C, xh);
        }
    }
}

// dweight / dbias: 32 columns x 32 slices of the partial rows a workgroup; slices are joined in order
template <class T>
__global__ __launch_bounds__(1024) void param_kernel(const float* __restrict__ part, void* dw, void* db, int nblk, int C, int w32) {
    __shared__ float s[32][33];
    const int half = blockIdx.y, col = threadIdx.x & 31, slice = threadIdx.x >> 5, c = blockIdx.x * 32 + col;
    void* out = half ? db : dw;
    if (!out) return;
    float sum = 0.f;
    if (c < C) {
#pragma unroll 8
        for (int k = slice; k < nblk; k += 32) sum += part[((long long)k * 2 + half) * C + c];
    }
    s[slice][col] = sum;
    __syncthreads();
    if (slice == 0 && c < C) {
        double t = 0.0;
        for (int k = 0; k < 32; ++k) t += (double)s[k][col];
        if (w32) reinterpret_cast<float*>(out)[c] = (float)t;
        else reinterpret_cast<T*>(out)[c] = (T)(float)t;
    }
}

// lanes a row and accesses a lane: the fewest lanes that hold the row in at most four accesses up to a wave, else a workgroup
template <class F> int by_width(int acc, F f) {       // acc: 16-byte accesses of a row
    if (acc <= 4) return f(std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{});
    if (acc <= 16) return f(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{});
    if (acc <= 64) return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
    if (acc <= 128) return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
    if (acc <= 256) return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
    if (acc <= 512) return f(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
    if (acc <= 1024) return f(std::integral_constant<int, 256>{}, std::integral_constant<int, 4>{});
    if (acc <= 2048) return f(std::integral_constant<int, 256>{}, std::integral_constant<int, 8>{});
    return f(std::integral_constant<int, 256>{}, std::integral_constant<int, 0>{});
}
static inline int rows_per_group(int acc) { return acc <= 4 ? 64 : acc <= 16 ? 16 : acc <= 256 ? 4 : 1; }

constexpr int FWD_BLOCKS = 2048, BWD_BLOCKS = 512;
template <class T> int fwd(const FwdParams& p, hipStream_t s) {
    const int acc = (p.C + VEC<T> - 1) / VEC<T>;
    const int grid = (int)std::min<long long>(FWD_BLOCKS, (p.rows + rows_per_group(acc) - 1) / rows_per_group(acc));
    return by_width(acc, [&](auto g, auto n) {
        if constexpr (n() == 0) hipLaunchKernelGGL((fwd_wide_kernel<T>), dim3(grid), dim3(256), 0, s, p);
        else hipLaunchKernelGGL((fwd_kernel<T, g(), n()>), dim3(grid), dim3(256), 0, s, p);
        DPC_LAUNCH_CHECK();
        return (int)DPC_OK;
    });
}

template <class T> int bwd(const BwdParams& p, void* dw, void* db, hipStream_t s) {
    const int acc = (p.C + VEC<T> - 1) / VEC<T>;
    const int grid = (int)std::min<long long>(BWD_BLOCKS, (p.rows + rows_per_group(acc) - 1) / rows_per_group(acc));
    const int rc = by_width(acc, [&](auto g, auto n) {
        if constexpr (n() == 0) hipLaunchKernelGGL((bwd_wide_kernel<T>), dim3(grid), dim3(256), 0, s, p);
        else hipLaunchKernelGGL((bwd_kernel<T, g(), n()>), dim3(grid), dim3(256), 0, s, p);
        DPC_LAUNCH_CHECK();
        return (int)DPC_OK;
    });
    if (rc != DPC_OK || !p.part) return rc;
    hipLaunchKernelGGL((param_kernel<T>), dim3((p.C + 31) / 32, 2), dim3(1024), 0, s, p.part, dw, db, grid, p.C, p.w32);
    DPC_LAUNCH_CHECK();
    return DPC_OK;
}

static int vector_rows(const void* a, const void* b, const void* c, long long sa, long long sb, int C, int es) {
    const size_t bits = (size_t)a | (size_t)b | (size_t)c | (size_t)(sa * es) | (size_t)(sb * es) | (size_t)((long long)C * es);
    return bits % 16 == 0;
}

}  // namespace seqnorm
}  // namespace dpc

using namespace dpc;
using namespace dpc::seqnorm;

extern "C" {

int dpc_seq_norm_fwd(const void* x, const void* weight, const void* bias, void* y, float* stats, int64_t rows, int C,
                     int64_t x_stride, float eps, int type, int wtype, dpc_stream_t stream) {
    DPC_REQUIRE(type >= DPC_SEQ_F32 && type <= DPC_SEQ_BF16, "seq_norm: unknown element type");
    DPC_REQUIRE(wtype == DPC_SEQ_F32 || wtype == type, "seq_norm: weight and bias are fp32 or of the element type");
    DPC_REQUIRE(rows >= 0 && C >= 1 && eps > 0.f, "seq_norm: rows >= 0, C >= 1, eps > 0");
    if (rows == 0) return DPC_OK;
    DPC_REQUIRE(x && y && stats && (rows == 1 || x_stride >= C), "seq_norm: null argument or overlapping rows");
    hipStream_t s = (hipStream_t)stream;
    const int es = type == DPC_SEQ_F32 ? 4 : 2;
    const FwdParams p{x, weight, bias, y, stats, rows, x_stride, C, wtype == DPC_SEQ_F32, vector_rows(x, y, nullptr, x_stride, 0, C, es), eps};
    ProfScope prof(PROF_LN, 0, 2.0 * (double)rows * C * es, s);
    return type == DPC_SEQ_F32 ? fwd<float>(p, s) : type == DPC_SEQ_F16 ? fwd<_Float16>(p, s) : fwd<__bf16>(p, s);
}

size_t dpc_seq_norm_bwd_workspace_bytes(int64_t rows, int C) {
    if (rows < 1 || C < 1) return 0;
    return (size_t)std::min<long long>(BWD_BLOCKS, rows) * 2 * (size_t)C * sizeof(float) + 256;
}

int dpc_seq_norm_bwd(const void* dy, const void* x, const float* stats, const void* weight, void* dx, void* dweight, void* dbias,
                     int64_t rows, int C, int64_t dy_stride, int64_t x_stride, int type, int wtype, void* ws, size_t ws_bytes,
                     dpc_stream_t stream) {
    DPC_REQUIRE(type >= DPC_SEQ_F32 && type <= DPC_SEQ_BF16, "seq_norm_bwd: unknown element type");
    DPC_REQUIRE(wtype == DPC_SEQ_F32 || wtype == type, "seq_norm_bwd: weight and bias are fp32 or of the element type");
    DPC_REQUIRE(rows >= 1 && C >= 1, "seq_norm_bwd: rows >= 1, C >= 1");
    DPC_REQUIRE(dy && x && stats && dx && (rows == 1 || (x_stride >= C && (dy_stride >= C || dy_stride == 0))), "seq_norm_bwd: null argument or overlapping rows");
    const bool sums = dweight || dbias;
    DPC_REQUIRE(!sums || (ws && ws_bytes >= dpc_seq_norm_bwd_workspace_bytes(rows, C)), "seq_norm_bwd: workspace too small");
    hipStream_t s = (hipStream_t)stream;
    const int es = type == DPC_SEQ_F32 ? 4 : 2;
    const BwdParams p{dy, x, weight, stats, dx, sums ? reinterpret_cast<float*>(align_up((size_t)ws, 256)) : nullptr, rows, dy_stride, x_stride, C,
                      wtype == DPC_SEQ_F32, vector_rows(dy, x, dx, dy_stride, x_stride, C, es)};
    ProfScope prof(PROF_LN, 0, 3.0 * (double)rows * C * es, s);
    return type == DPC_SEQ_F32 ? bwd<float>(p, dweight, dbias, s) : type == DPC_SEQ_F16 ? bwd<_Float16>(p, dweight, dbias, s) : bwd<__bf16>(p, dweight, dbias, s);
}

}  // extern "C"
