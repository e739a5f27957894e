// Layer norm over the last axis, forward and backward (include/dpc.h: dpc_seq_norm_*).
//   mu = sum x / C, var = sum (x - mu)^2 / C, s = (var + eps)^-1/2, xh = (x - mu) s, y = xh w + b
//   g = dy w, dx = s (g - mean(g) - xh mean(g xh)), dw = sum_rows dy xh, db = sum_rows dy
// Bound by bytes: the forward reads x and writes y, the backward reads x and dy and writes dx, each once.  A row lives in the registers
// of G lanes (4, 16, 64 or a whole workgroup; N accesses of 16 bytes a lane), so that the centred second sum of the variance -- no
// E[x^2] - mu^2 cancellation -- costs no second read.  Rows too wide for that (over 2048 accesses) are read again from L2.
// The backward pass keeps dw and db in registers over all rows of a group, adds the groups of a workgroup in LDS and writes one row of
// partial sums per workgroup; a second kernel adds those in fixed order (in fp32, the last 32 of a column in double).
// fp32 786432 x 64: forward 71 us (5.7 TB/s), backward 120 (5.0) and 7 for the sums; bf16 8191 x 4096: 23 (5.7), 47 (4.3; 42 on another card) and 5.
// Rows over 2048 accesses add dw and db in global memory, row by row, 16 bytes an element beside the row's own 12: fp32 4000 x 12000 forward 107 us, backward 481.
#include <algorithm>
#include <initializer_list>
#include <type_traits>
#include <utility>

#include "common.h"

namespace dpc {
namespace seqnorm {

template <class T> constexpr int VEC = 16 / (int)sizeof(T);
template <class T, int E> struct Pack { typedef T type __attribute__((ext_vector_type(E))); };

// Element e of access n of a lane.  VECT: rows start on 16 bytes and hold whole accesses; a lane has 16 consecutive bytes.  Otherwise: one
// element at a time, consecutive lanes on consecutive elements.
template <class T, int G, bool VECT> __device__ __forceinline__ int at(int lane, int n, int e) {
    return VECT ? (n * G + lane) * VEC<T> + e : n * G * VEC<T> + e * G + lane;
}

// The elements of P (T, or fp32 parameters) that a lane holds, as they lie in memory; `none` past the row's end
template <class T, class P, int G, int N, bool VECT> struct Held {
    typedef typename Pack<P, VEC<T>>::type Q;
    Q v[N];
    __device__ __forceinline__ void load(const P* __restrict__ row, int lane, int C, float none) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if (VECT) {
                const int c = at<T, G, VECT>(lane, n, 0);
                if (c < C) { v[n] = *reinterpret_cast<const Q*>(row + c); continue; }
            }
#pragma unroll
            for (int e = 0; e < VEC<T>; ++e) {
                const int c = at<T, G, VECT>(lane, n, e);
                v[n][e] = !VECT && c < C ? row[c] : (P)none;
            }
        }
    }
    // A row that is on its way while another is worked on: ask() reads something in every lane and settled() puts zeros past the row's end.  (With the
    // choice at the load, the compiler copies what was loaded, and waits for it, right behind the load: bf16 8191 x 4096 backward 14 % slower.  Rows of
    // a wave or less, of which thousands are at work, lose by ask(): fp32 786432 x 64 7 %.)
    __device__ __forceinline__ void ask(const P* __restrict__ row, int lane, int C) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if (VECT) {
                const int c = at<T, G, VECT>(lane, n, 0);
                v[n] = *reinterpret_cast<const Q*>(row + (c < C ? c : 0));
                continue;
            }
#pragma unroll
            for (int e = 0; e < VEC<T>; ++e) { const int c = at<T, G, VECT>(lane, n, e); v[n][e] = row[c < C ? c : 0]; }
        }
    }
    __device__ __forceinline__ Held settled(int lane, int C) const {
        Held r;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if (VECT) {
                const uint4 w = __builtin_bit_cast(uint4, v[n]);
                const unsigned m = at<T, G, VECT>(lane, n, 0) < C ? ~0u : 0u;
                r.v[n] = __builtin_bit_cast(Q, uint4{w.x & m, w.y & m, w.z & m, w.w & m});
                continue;
            }
#pragma unroll
            for (int e = 0; e < VEC<T>; ++e) r.v[n][e] = at<T, G, VECT>(lane, n, e) < C ? v[n][e] : (P)0.f;
        }
        return r;
    }
    __device__ __forceinline__ void fill(float x) {
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < VEC<T>; ++e) v[n][e] = (P)x;
    }
};

template <class T, int G, bool VECT> __device__ __forceinline__ void store(T* __restrict__ row, int lane, int n, int C, const float (&v)[VEC<T>]) {
    typedef typename Pack<T, VEC<T>>::type Q;
    if (VECT) {
        const int c = at<T, G, VECT>(lane, n, 0);
        if (c < C) {
            Q q;
#pragma unroll
            for (int e = 0; e < VEC<T>; ++e) q[e] = (T)v[e];
            *reinterpret_cast<Q*>(row + c) = q;
        }
    } else {
#pragma unroll
        for (int e = 0; e < VEC<T>; ++e) { const int c = at<T, G, VECT>(lane, n, e); if (c < C) row[c] = (T)v[e]; }
    }
}

// Sums of a and b over the G lanes of a group.  A group that is a whole workgroup (256 to 1024) meets in LDS; `turn` alternates between two slots, so one
// barrier a call is enough.  (Every thread of the workgroup makes every call.)
template <int G> __device__ __forceinline__ void group_sum(float& a, float& b, float2 (*s_red)[16], int& turn) {
#pragma unroll
    for (int x = (G < 64 ? G : 64) / 2; x; x >>= 1) { a += __shfl_xor(a, x, 64); b += __shfl_xor(b, x, 64); }
    if (G > 64) {
        if ((threadIdx.x & 63) == 0) s_red[turn][threadIdx.x >> 6] = float2{a, b};
        __syncthreads();
        if (G <= 256) {
            a = b = 0.f;
#pragma unroll
            for (int w = 0; w < G / 64; ++w) { a += s_red[turn][w].x; b += s_red[turn][w].y; }
        } else {                                                     // (a lane a wave: reading all of 16 would take 32 registers)
            const float2 z = s_red[turn][threadIdx.x & (G / 64 - 1)];
            a = z.x;
            b = z.y;
#pragma unroll
            for (int x = G / 128; x; x >>= 1) { a += __shfl_xor(a, x, 64); b += __shfl_xor(b, x, 64); }
        }
        turn ^= 1;
    }
}

struct FwdParams {
    const void *x, *w, *b;
    void* y;
    float* stats;
    long long rows, xs;
    int C, vec;
    float eps;
};

template <class T, class P, int G, int N, bool VECT, int THREADS>
__global__ __launch_bounds__(THREADS) void fwd_kernel(const FwdParams p) {
    __shared__ float2 s_red[2][16];
    constexpr int V = VEC<T>, R = THREADS / G;
    const int lane = threadIdx.x & (G - 1);
    int turn = 0;
    const float inv_c = 1.f / (float)p.C;
    Held<T, P, G, N, VECT> w, b;
    if (p.w) w.load(reinterpret_cast<const P*>(p.w), lane, p.C, 0.f); else w.fill(1.f);
    if (p.b) b.load(reinterpret_cast<const P*>(p.b), lane, p.C, 0.f); else b.fill(0.f);
    const long long step = (long long)gridDim.x * R;
    long long r = (long long)blockIdx.x * R + threadIdx.x / G;
    const T* x = reinterpret_cast<const T*>(p.x);
    Held<T, T, G, N, VECT> next;
    next.load(x + min(r, p.rows - 1) * p.xs, lane, p.C, 0.f);
    for (long long r0 = (long long)blockIdx.x * R; r0 < p.rows; r0 += step, r += step) {      // (uniform over the workgroup)
        Held<T, T, G, N, VECT> cur = next;
        if (r0 + step < p.rows) next.load(x + min(r + step, p.rows - 1) * p.xs, lane, p.C, 0.f);
        float v[N][V], sum = 0.f, none = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < V; ++e) { v[n][e] = (float)cur.v[n][e]; sum += v[n][e]; }
        group_sum<G>(sum, none, s_red, turn);
        const float mu = sum * inv_c;
        sum = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[n][e] -= mu;
                if (at<T, G, VECT>(lane, n, e) < p.C) sum = __builtin_fmaf(v[n][e], v[n][e], sum);
            }
        group_sum<G>(sum, none, s_red, turn);
        const float rstd = 1.f / sqrtf(sum * inv_c + p.eps);
        if (r < p.rows) {
            T* y = reinterpret_cast<T*>(p.y) + r * (long long)p.C;
#pragma unroll
            for (int n = 0; n < N; ++n) {
#pragma unroll
                for (int e = 0; e < V; ++e) v[n][e] = __builtin_fmaf(v[n][e] * rstd, (float)w.v[n][e], (float)b.v[n][e]);
                store<T, G, VECT>(y, lane, n, p.C, v[n]);
            }
            if (lane == 0) *reinterpret_cast<float2*>(p.stats + 2 * r) = float2{mu, rstd};
        }
    }
}

// rows wider than 2048 accesses: one workgroup a row, three reads of x (the later two from L2)
template <class T, class P, bool VECT>
__global__ __launch_bounds__(256) void fwd_wide_kernel(const FwdParams p) {
    __shared__ float2 s_red[2][16];
    constexpr int V = VEC<T>, S = 256 * V;
    const int lane = threadIdx.x;
    int turn = 0;
    const float inv_c = 1.f / (float)p.C;
    for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* x = reinterpret_cast<const T*>(p.x) + r * p.xs;
        Held<T, T, 256, 1, VECT> h;
        float sum = 0.f, none = 0.f;
        for (int c0 = 0; c0 < p.C; c0 += S) {
            h.load(x + c0, lane, p.C - c0, 0.f);
#pragma unroll
            for (int e = 0; e < V; ++e) sum += (float)h.v[0][e];
        }
        group_sum<256>(sum, none, s_red, turn);
        const float mu = sum * inv_c;
        sum = 0.f;
        for (int c0 = 0; c0 < p.C; c0 += S) {
            h.load(x + c0, lane, p.C - c0, 0.f);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = (float)h.v[0][e] - mu;
                if (c0 + at<T, 256, VECT>(lane, 0, e) < p.C) sum = __builtin_fmaf(d, d, sum);
            }
        }
        group_sum<256>(sum, none, s_red, turn);
        const float rstd = 1.f / sqrtf(sum * inv_c + p.eps);
        T* y = reinterpret_cast<T*>(p.y) + r * (long long)p.C;
        for (int c0 = 0; c0 < p.C; c0 += S) {
            Held<T, P, 256, 1, VECT> w, b;
            h.load(x + c0, lane, p.C - c0, 0.f);
            if (p.w) w.load(reinterpret_cast<const P*>(p.w) + c0, lane, p.C - c0, 0.f); else w.fill(1.f);
            if (p.b) b.load(reinterpret_cast<const P*>(p.b) + c0, lane, p.C - c0, 0.f); else b.fill(0.f);
            float v[V];
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = __builtin_fmaf(((float)h.v[0][e] - mu) * rstd, (float)w.v[0][e], (float)b.v[0][e]);
            store<T, 256, VECT>(y + c0, lane, 0, p.C - c0, v);
        }
        if (lane == 0) *reinterpret_cast<float2*>(p.stats + 2 * r) = float2{mu, rstd};
    }
}

struct BwdParams {
    const void *dy, *x, *w;
    const float* stats;
    void *dx, *dw, *db;        // dw, db: written by the kernel itself when it is one workgroup (part null)
    float* part;               // [gridDim.x][2][C] sums of dy xh and dy
    long long rows, dys, xs;
    int C, vec, sums;
};

template <class P> __device__ __forceinline__ void put_param(void* dst, int c, float v) { if (dst) reinterpret_cast<P*>(dst)[c] = (P)v; }

template <class T, class P, int G, int N, bool VECT, int THREADS>
__global__ __launch_bounds__(THREADS) void bwd_kernel(const BwdParams p) {
    constexpr int V = VEC<T>, R = THREADS / G;
    constexpr bool WG_ROW = G > 64;                                   // few rows at once: the next one has to be on its way
    __shared__ float2 s_red[2][16];
    __shared__ float s_sum[R > 1 ? THREADS * N * V : 1];
    const int lane = threadIdx.x & (G - 1), grp = threadIdx.x / G;
    int turn = 0;
    const float inv_c = 1.f / (float)p.C;
    float dw[N][V], db[N][V];
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int e = 0; e < V; ++e) dw[n][e] = db[n][e] = 0.f;
    Held<T, P, G, N, VECT> w;
    if (p.w) w.load(reinterpret_cast<const P*>(p.w), lane, p.C, 0.f); else w.fill(1.f);
    const T* x = reinterpret_cast<const T*>(p.x);
    const T* dy = reinterpret_cast<const T*>(p.dy);
    const long long step = (long long)gridDim.x * R;
    long long r = (long long)blockIdx.x * R + grp;
    Held<T, T, G, N, VECT> nx, ny;
    float2 ns;
    auto fetch = [&](long long row) {
        row = min(row, p.rows - 1);
        if (WG_ROW) {
            nx.ask(x + row * p.xs, lane, p.C);
            ny.ask(dy + row * p.dys, lane, p.C);
        } else {
            nx.load(x + row * p.xs, lane, p.C, 0.f);
            ny.load(dy + row * p.dys, lane, p.C, 0.f);
        }
        ns = *reinterpret_cast<const float2*>(p.stats + 2 * row);
    };
    fetch(r);
    for (long long r0 = (long long)blockIdx.x * R; r0 < p.rows; r0 += step, r += step) {
        Held<T, T, G, N, VECT> hx = WG_ROW ? nx.settled(lane, p.C) : nx, hy = WG_ROW ? ny.settled(lane, p.C) : ny;
        const float mu = ns.x, rstd = ns.y;
        if (r0 + step < p.rows) fetch(r + step);
        float a = 0.f, b = 0.f;
        // (past the row's end xh is 0 as dy is: (0 - mu) rstd may leave fp32's range where the row's own xh do not, and 0 * inf would reach every dx)
        auto xhat = [&](int n, int e) { return ((float)hx.v[n][e] - mu) * (at<T, G, VECT>(lane, n, e) < p.C ? rstd : 0.f); };
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float xh = xhat(n, e);
                float g = (float)hy.v[n][e];                         // (0 past the row's end)
                if (r >= p.rows) g = 0.f;                            // (a group without a row reads the last one again)
                dw[n][e] = __builtin_fmaf(g, xh, dw[n][e]);
                db[n][e] += g;
                g *= (float)w.v[n][e];
                a += g;
                b = __builtin_fmaf(g, xh, b);
            }
        group_sum<G>(a, b, s_red, turn);
        a *= inv_c;
        b *= inv_c;
        if (r < p.rows) {
            T* dx = reinterpret_cast<T*>(p.dx) + r * (long long)p.C;
#pragma unroll
            for (int n = 0; n < N; ++n) {
                float v[V];
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] = rstd * ((float)hy.v[n][e] * (float)w.v[n][e] - __builtin_fmaf(xhat(n, e), b, a));
                store<T, G, VECT>(dx, lane, n, p.C, v);
            }
        }
    }
    if (!p.sums) return;
    // the groups of the workgroup are added in order, first dw, then db
    float* part = p.part ? p.part + (long long)blockIdx.x * 2 * p.C : nullptr;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        if (R > 1) {
            __syncthreads();
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int e = 0; e < V; ++e) s_sum[(grp * N * V + n * V + e) * G + lane] = half ? db[n][e] : dw[n][e];
            __syncthreads();
        }
        constexpr int W = G * N * V;                                 // columns a group holds: index (n V + e) G + lane
        for (int i = threadIdx.x; i < W; i += THREADS) {
            float sum = 0.f;
            if (R > 1) {
#pragma unroll 8
                for (int q = 0; q < R; ++q) sum += s_sum[q * W + i];
            }
            const int c = at<T, G, VECT>(i % G, i / G / V, i / G % V);
            if (R == 1) {                                            // (i = (n V + e) G + thread: this thread's own)
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int e = 0; e < V; ++e) if (n * V + e == i / G) sum = half ? db[n][e] : dw[n][e];
            }
            if (c >= p.C) continue;
            if (part) part[half * p.C + c] = sum;
            else put_param<P>(half ? p.db : p.dw, c, sum);
        }
    }
}

template <class T, class P, bool VECT>
__global__ __launch_bounds__(256) void bwd_wide_kernel(const BwdParams p) {
    __shared__ float2 s_red[2][16];
    constexpr int V = VEC<T>, S = 256 * V;
    const int lane = threadIdx.x;
    int turn = 0;
    const float inv_c = 1.f / (float)p.C;
    float* part = p.sums ? p.part + (long long)blockIdx.x * 2 * p.C : nullptr;
    bool first = true;
    for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* x = reinterpret_cast<const T*>(p.x) + r * p.xs;
        const T* dy = reinterpret_cast<const T*>(p.dy) + r * p.dys;
        const float mu = p.stats[2 * r], rstd = p.stats[2 * r + 1];
        Held<T, T, 256, 1, VECT> hx, hy;
        Held<T, P, 256, 1, VECT> w;
        w.fill(1.f);
        float a = 0.f, b = 0.f;
        for (int c0 = 0; c0 < p.C; c0 += S) {
            hx.load(x + c0, lane, p.C - c0, 0.f);
            hy.load(dy + c0, lane, p.C - c0, 0.f);
            if (p.w) w.load(reinterpret_cast<const P*>(p.w) + c0, lane, p.C - c0, 0.f);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int c = c0 + at<T, 256, VECT>(lane, 0, e);
                if (c >= p.C) continue;
                const float xh = ((float)hx.v[0][e] - mu) * rstd, g = (float)hy.v[0][e];
                if (part) {                                          // (this thread's own columns: no other touches them)
                    part[c] = (first ? 0.f : part[c]) + g * xh;
                    part[p.C + c] = (first ? 0.f : part[p.C + c]) + g;
                }
                a += g * (float)w.v[0][e];
                b = __builtin_fmaf(g * (float)w.v[0][e], xh, b);
            }
        }
        first = false;
        group_sum<256>(a, b, s_red, turn);
        a *= inv_c;
        b *= inv_c;
        T* dx = reinterpret_cast<T*>(p.dx) + r * (long long)p.C;
        for (int c0 = 0; c0 < p.C; c0 += S) {
            hx.load(x + c0, lane, p.C - c0, 0.f);
            hy.load(dy + c0, lane, p.C - c0, 0.f);
            if (p.w) w.load(reinterpret_cast<const P*>(p.w) + c0, lane, p.C - c0, 0.f);
            float v[V];
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = rstd * ((float)hy.v[0][e] * (float)w.v[0][e] - __builtin_fmaf(((float)hx.v[0][e] - mu) * rstd, b, a));
            store<T, 256, VECT>(dx + c0, lane, 0, p.C - c0, v);
        }
    }
}

// dweight / dbias: 32 columns x 32 slices of the partial rows a workgroup, which goes on by whole grids (a launch holds fewer than 2^32 threads); slices
// are joined in order
constexpr int PARAM_BLOCKS = 1 << 16;
template <class P>
__global__ __launch_bounds__(1024) void param_kernel(const float* __restrict__ part, void* dw, void* db, int nblk, int C) {
    __shared__ float s[32][33];
    const int half = blockIdx.y, col = threadIdx.x & 31, slice = threadIdx.x >> 5;
    void* out = half ? db : dw;
    if (!out) return;
    for (int c0 = blockIdx.x * 32; c0 < C; c0 += gridDim.x * 32) {
        const int c = c0 + col;
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
            put_param<P>(out, c, (float)t);
        }
        __syncthreads();
    }
}

// Lanes a row (G) and accesses a lane (N) by the row's 16-byte accesses: the fewest lanes that hold it in at most four accesses up to a wave
// -- no barrier -- else a workgroup.  More accesses a lane cost registers, that is waves, that is loads in flight: bf16 rows of 4096 forward in
// one wave of 8 accesses take 1.8 times as long as in four waves of 2.  The backward pass holds four times as much a lane and goes to workgroups of one
// access a lane earlier: bf16 8191 x 8192 in four accesses 119 us, in one 97; 30000 x 2048 84 and 80.
template <int A, int B> using Shape = std::pair<std::integral_constant<int, A>, std::integral_constant<int, B>>;
template <bool BWD, class F> int by_width(int acc, F f) {
    if (acc <= 4) return f(Shape<4, 1>{});
    if (acc <= 16) return f(Shape<16, 1>{});
    if (acc <= 64) return f(Shape<64, 1>{});
    if (acc <= 128) return f(Shape<64, 2>{});
    if (acc <= 256) return f(Shape<BWD ? 256 : 64, BWD ? 1 : 4>{});
    if (acc <= 512) return f(Shape<BWD ? 512 : 256, BWD ? 1 : 2>{});
    if (acc <= 1024) return f(Shape<BWD ? 1024 : 256, BWD ? 1 : 4>{});
    if (acc <= 2048) return f(Shape<1024, 2>{});
    return f(Shape<256, 0>{});
}

constexpr int FWD_BLOCKS = 2048;
constexpr int MAX_C = 1 << 30;                // columns are counted in 32 bits, a step of 2048 accesses past the last one included
// Workgroups of the backward pass: each writes one row of partial sums (8 C bytes, read once more), which may cost some 10 % of the rows' own traffic,
// but two workgroups a CU are there in any case.
static int bwd_blocks(long long rows, int es) { return (int)std::min(rows, std::min(2048ll, std::max(512ll, rows * es / 64))); }
constexpr long long ONE_BLOCK = 32768;       // elements that one workgroup of 1024 threads takes alone: the sums then need no second launch

static bool one_block(long long rows, int C, int es) { return rows * C <= ONE_BLOCK && (C * es + 15) / 16 <= 64; }

template <class T, class P, bool VECT> int fwd(const FwdParams& p, hipStream_t s) {
    const int acc = (p.C + VEC<T> - 1) / VEC<T>;
    return by_width<false>(acc, [&](auto shape) {
        constexpr int G = decltype(shape.first)::value, N = decltype(shape.second)::value;
        constexpr int THREADS = G > 256 ? G : 256, R = THREADS / G;
        const int grid = (int)std::min<long long>(FWD_BLOCKS, (p.rows + R - 1) / R);
        if constexpr (N == 0) hipLaunchKernelGGL((fwd_wide_kernel<T, P, VECT>), dim3(grid), dim3(256), 0, s, p);
        else hipLaunchKernelGGL((fwd_kernel<T, P, G, N, VECT, THREADS>), dim3(grid), dim3(THREADS), 0, s, p);
        DPC_LAUNCH_CHECK();
        return (int)DPC_OK;
    });
}

template <class T, class P, bool VECT> int bwd(const BwdParams& p, hipStream_t s) {
    const int acc = (p.C + VEC<T> - 1) / VEC<T>;
    return by_width<true>(acc, [&](auto shape) {
        constexpr int G = decltype(shape.first)::value, N = decltype(shape.second)::value;
        if constexpr (G <= 64 && N == 1) {
            if (p.sums && !p.part) {
                hipLaunchKernelGGL((bwd_kernel<T, P, G, N, VECT, 1024>), dim3(1), dim3(1024), 0, s, p);
                DPC_LAUNCH_CHECK();
                return (int)DPC_OK;
            }
        }
        constexpr int THREADS = G > 256 ? G : 256, R = THREADS / G;
        const int grid = (int)std::min<long long>(bwd_blocks(p.rows, sizeof(T)), (p.rows + R - 1) / R);
        if constexpr (N == 0) hipLaunchKernelGGL((bwd_wide_kernel<T, P, VECT>), dim3(grid), dim3(256), 0, s, p);
        else hipLaunchKernelGGL((bwd_kernel<T, P, G, N, VECT, THREADS>), dim3(grid), dim3(THREADS), 0, s, p);
        DPC_LAUNCH_CHECK();
        if (!p.sums) return (int)DPC_OK;
        hipLaunchKernelGGL((param_kernel<P>), dim3(std::min((p.C + 31) / 32, PARAM_BLOCKS), 2), dim3(1024), 0, s, p.part, p.dw, p.db, grid, p.C);
        DPC_LAUNCH_CHECK();
        return (int)DPC_OK;
    });
}

template <class Prm, class F> int by_type(const Prm& p, int type, int wtype, F f) {
    auto v = [&](auto t, auto w) { return p.vec ? f(t, w, std::true_type{}) : f(t, w, std::false_type{}); };
    if (type == DPC_SEQ_F32) return v(float{}, float{});
    if (type == DPC_SEQ_F16) return wtype == DPC_SEQ_F32 ? v(_Float16{}, float{}) : v(_Float16{}, _Float16{});
    return wtype == DPC_SEQ_F32 ? v(__bf16{}, float{}) : v(__bf16{}, __bf16{});
}

// (parameters of fp32 beside a 16-bit x are read 32 bytes at a time)
static int vector_rows(std::initializer_list<const void*> ptrs, long long sa, long long sb, int C, int es, const void* w, const void* b, int wes) {
    size_t bits = (size_t)(sa * es) | (size_t)(sb * es) | (size_t)((long long)C * es);
    for (const void* q : ptrs) bits |= (size_t)q;
    return bits % 16 == 0 && ((size_t)w | (size_t)b) % (16 / es * wes) == 0;
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
    DPC_REQUIRE(rows >= 0 && C >= 1 && C <= MAX_C && eps > 0.f, "seq_norm: rows >= 0, 1 <= C <= 2^30, eps > 0");
    if (rows == 0) return DPC_OK;
    DPC_REQUIRE(x && y && stats && (rows == 1 || x_stride >= C), "seq_norm: null argument or overlapping rows");
    hipStream_t s = (hipStream_t)stream;
    const int es = type == DPC_SEQ_F32 ? 4 : 2;
    const FwdParams p{x, weight, bias, y, stats, rows, x_stride, C, vector_rows({x, y}, x_stride, 0, C, es, weight, bias, wtype == DPC_SEQ_F32 ? 4 : 2), eps};
    ProfScope prof(PROF_LN, 0, 2.0 * (double)rows * C * es, s);
    return by_type(p, type, wtype, [&](auto t, auto w, auto v) { return fwd<decltype(t), decltype(w), decltype(v)::value>(p, s); });
}

size_t dpc_seq_norm_bwd_workspace_bytes(int64_t rows, int C, int type) {
    if (rows < 1 || C < 1 || C > MAX_C || one_block(rows, C, type == DPC_SEQ_F32 ? 4 : 2)) return 0;
    return (size_t)bwd_blocks(rows, type == DPC_SEQ_F32 ? 4 : 2) * 2 * (size_t)C * sizeof(float) + 256;
}

int dpc_seq_norm_bwd(const void* dy, const void* x, const float* stats, const void* weight, void* dx, void* dweight, void* dbias,
                     int64_t rows, int C, int64_t dy_stride, int64_t x_stride, int type, int wtype, void* ws, size_t ws_bytes,
                     dpc_stream_t stream) {
    DPC_REQUIRE(type >= DPC_SEQ_F32 && type <= DPC_SEQ_BF16, "seq_norm_bwd: unknown element type");
    DPC_REQUIRE(wtype == DPC_SEQ_F32 || wtype == type, "seq_norm_bwd: weight and bias are fp32 or of the element type");
    DPC_REQUIRE(rows >= 1 && C >= 1 && C <= MAX_C, "seq_norm_bwd: rows >= 1, 1 <= C <= 2^30");
    DPC_REQUIRE(dy && x && stats && dx && (rows == 1 || (x_stride >= C && (dy_stride >= C || dy_stride == 0))), "seq_norm_bwd: null argument or overlapping rows");
    const int sums = dweight || dbias, es = type == DPC_SEQ_F32 ? 4 : 2;
    const size_t need = sums ? dpc_seq_norm_bwd_workspace_bytes(rows, C, type) : 0;
    DPC_REQUIRE(need == 0 || (ws && ws_bytes >= need), "seq_norm_bwd: workspace too small");
    hipStream_t s = (hipStream_t)stream;
    const BwdParams p{dy, x, weight, stats, dx, dweight, dbias, need ? reinterpret_cast<float*>(align_up((size_t)ws, 256)) : nullptr, rows, dy_stride, x_stride, C,
                      vector_rows({dy, x, dx}, dy_stride, x_stride, C, es, weight, nullptr, wtype == DPC_SEQ_F32 ? 4 : 2), sums};
    ProfScope prof(PROF_LN, 0, 3.0 * (double)rows * C * es, s);
    return by_type(p, type, wtype, [&](auto t, auto w, auto v) { return bwd<decltype(t), decltype(w), decltype(v)::value>(p, s); });
}

}  // extern "C"
