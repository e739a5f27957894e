// Rotary positions (include/dpc.h: dpc_seq_rotary): pair (a, b) of a head at position p becomes (a cos t - b sin t, a sin t + b cos t)
// with (cos, sin) = table[p][pair]; the gradient is the transpose (sin -> -sin), so both directions are this kernel.
// Bound by bytes: every element is read and written once.  A thread owns one chunk of a token's head and walks over heads with the chunk's cosines in
// registers.  Interleaved: a chunk is 16 bytes of pairs, or of the pass-through part.  Half layout: a chunk is any 16 bytes of the head, the lanes of a
// head read it in one piece, and the pair's other halves come from the lane that has them -- were they loaded, every line of memory would be touched by
// two loads and two stores (2 x 8192 tokens, 40 heads of 128, 96 of them turned, bf16: 81 -> 64 us).  Rows that do not start on 16 bytes, or halves that
// do not, go one pair at a time.  A copy's rate: 5.3 TB/s there, 5.2 for fp32 1536 x 32 tokens, 16 heads of 32 (39 us).
#include <algorithm>

#include "seq_div.h"

namespace dpc {
namespace seqrot {

struct Ten { char* p; long long b, t, h; };      // strides in elements

struct Params {
    Ten xq, xk, yq, yk;
    const float* table;
    const long long* positions;
    long long pos_b, start, max_pos;
    int total, heads, all, D, R, interleaved, rot_items, per_wg, work;
    Div tokens, items, per_token, groups;
    float sign;
};

template <class Q> __device__ __forceinline__ Q from_lane(const Q& v, int lane) {           // 16 bytes
    const uint4 w = __builtin_bit_cast(uint4, v);
    return __builtin_bit_cast(Q, uint4{(unsigned)__shfl((int)w.x, lane, 64), (unsigned)__shfl((int)w.y, lane, 64), (unsigned)__shfl((int)w.z, lane, 64), (unsigned)__shfl((int)w.w, lane, 64)});
}

// Half layout.  HEADS heads of one token: their loads are all in flight before the first is used.  The lanes of a row are in one wave: per_wg rows of
// (token, group of heads) a wave.
template <class T, int HEADS>
__global__ __launch_bounds__(256) void rotary_half_kernel(const Params p) {
    constexpr int V = 16 / (int)sizeof(T);
    typedef T Q __attribute__((ext_vector_type(V)));
    const unsigned lane = threadIdx.x & 63, wr = p.items(lane), it = lane - wr * p.items.d, row = (blockIdx.x * 4 + threadIdx.x / 64) * p.per_wg + wr;
    const bool turn = (int)it < p.rot_items;
    if (wr >= (unsigned)p.per_wg || row >= (unsigned)p.work) return;
    const unsigned n = p.groups(row), hg = row - n * p.groups.d, b = p.tokens(n), t = n - b * p.tokens.d;
    const int c0 = it * V, half = p.rot_items / 2;
    const bool second = (int)it >= half;
    const int mate = turn ? lane + (second ? -half : half) : lane;   // (that lane has the same row: both are active, or neither)
    float cs[V], sn[V];
#pragma unroll
    for (int k = 0; k < V; ++k) { cs[k] = 1.f; sn[k] = 0.f; }
    if (turn) {
        const long long pos = p.positions ? p.positions[b * p.pos_b + t] : p.start + t;
        const bool ok = pos >= 0 && pos < p.max_pos;
        const float2* tab = reinterpret_cast<const float2*>(p.table) + (ok ? pos : 0) * (p.R / 2) + (second ? c0 - p.R / 2 : c0);
        const float sign = second ? p.sign : -p.sign;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float2 z = tab[k];
            cs[k] = ok ? z.x : __builtin_nanf("");
            sn[k] = ok ? z.y * sign : __builtin_nanf("");
        }
    }
    Q q[HEADS];
    T* dst[HEADS];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        const int hd = hg + i * p.groups.d;
        dst[i] = nullptr;
        if (hd >= p.all) continue;
        const bool isq = hd < p.heads;
        const Ten& X = isq ? p.xq : p.xk;
        const Ten& Y = isq ? p.yq : p.yk;
        const int h = isq ? hd : hd - p.heads;
        q[i] = *reinterpret_cast<const Q*>(reinterpret_cast<const T*>(X.p) + b * X.b + t * X.t + h * X.h + c0);
        dst[i] = reinterpret_cast<T*>(Y.p) + b * Y.b + t * Y.t + h * Y.h + c0;
    }
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        if (!dst[i]) continue;
        const Q u = from_lane(q[i], mate);
        if (turn) {
#pragma unroll
            for (int k = 0; k < V; ++k) q[i][k] = (T)((float)q[i][k] * cs[k] + (float)u[k] * sn[k]);
        }
        *reinterpret_cast<Q*>(dst[i]) = q[i];
    }
}

// Interleaved layout by chunks (V > 1), and either layout one pair at a time (V = 1).  HEADS as above.
template <class T, int V, int HEADS>
__global__ __launch_bounds__(256) void rotary_kernel(const Params p) {
    typedef T Q __attribute__((ext_vector_type(V)));
    constexpr int NP = V > 1 ? V : 1, PAIR = V > 1 ? V : 2;          // pairs of a chunk at most; elements of an interleaved chunk
    const unsigned w = threadIdx.x + blockIdx.y * 256;
    if (w >= (unsigned)p.work) return;
    const unsigned lt = p.per_token(w), in = w - lt * p.per_token.d, hg = p.items(in), it = in - hg * p.items.d;
    const unsigned n = blockIdx.x * p.per_wg + lt;
    if (n >= (unsigned)p.total) return;
    const unsigned b = p.tokens(n), t = n - b * p.tokens.d;
    const bool turn = (int)it < p.rot_items;
    const int c0 = !turn ? p.R + ((int)it - p.rot_items) * V : p.interleaved ? it * PAIR : it;
    const int other = V > 1 || !turn ? 0 : p.interleaved ? 1 : p.R / 2;               // distance to the pair's second half
    float cs[NP], sn[NP];
#pragma unroll
    for (int k = 0; k < NP; ++k) { cs[k] = 1.f; sn[k] = 0.f; }
    if (turn) {
        const long long pos = p.positions ? p.positions[b * p.pos_b + t] : p.start + t;
        const bool ok = pos >= 0 && pos < p.max_pos;
        const int i0 = it * (PAIR / 2);
        const float2* tab = reinterpret_cast<const float2*>(p.table) + (ok ? pos : 0) * (p.R / 2) + i0;
#pragma unroll
        for (int k = 0; k < NP; ++k)
            if (k < PAIR / 2) {
                const float2 z = tab[k];
                cs[k] = ok ? z.x : __builtin_nanf("");
                sn[k] = ok ? z.y * p.sign : __builtin_nanf("");
            }
    }
    Q q[HEADS], u[HEADS];
    T* dst[HEADS];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        const int hd = hg + i * p.groups.d;
        dst[i] = nullptr;
        if (hd >= p.all) continue;
        const bool isq = hd < p.heads;
        const Ten& X = isq ? p.xq : p.xk;
        const Ten& Y = isq ? p.yq : p.yk;
        const int h = isq ? hd : hd - p.heads;
        const T* x = reinterpret_cast<const T*>(X.p) + b * X.b + t * X.t + h * X.h + c0;
        dst[i] = reinterpret_cast<T*>(Y.p) + b * Y.b + t * Y.t + h * Y.h + c0;
        q[i] = *reinterpret_cast<const Q*>(x);
        u[i] = q[i];
        if (other) u[i] = *reinterpret_cast<const Q*>(x + other);
    }
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        if (!dst[i]) continue;
        if (turn && V > 1) {
#pragma unroll
            for (int k = 0; k < V / 2; ++k) {
                const float x = (float)q[i][2 * k], y = (float)q[i][(2 * k + 1) % V];
                q[i][2 * k] = (T)(x * cs[k] - y * sn[k]);
                q[i][(2 * k + 1) % V] = (T)(x * sn[k] + y * cs[k]);
            }
        } else if (turn) {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float x = (float)q[i][k], y = (float)u[i][k];
                q[i][k] = (T)(x * cs[k] - y * sn[k]);
                u[i][k] = (T)(x * sn[k] + y * cs[k]);
            }
        }
        *reinterpret_cast<Q*>(dst[i]) = q[i];
        if (other) *reinterpret_cast<Q*>(dst[i] + other) = u[i];
    }
}

constexpr unsigned MAX_GRID = 1u << 24;          // workgroups of 256 threads along an axis: a launch holds fewer than 2^32

static bool aligned(const dpc_seq_tensor& t, int es) {
    return !t.p || ((size_t)t.p | (size_t)(t.stride_b * es) | (size_t)(t.stride_t * es) | (size_t)(t.stride_h * es)) % 16 == 0;
}

static bool same(const dpc_seq_tensor& a, const dpc_seq_tensor& b) {
    return a.p == b.p && a.stride_b == b.stride_b && a.stride_t == b.stride_t && a.stride_h == b.stride_h;
}

template <class T> int run(const dpc_seq_rotary* a, hipStream_t s) {
    const int es = (int)sizeof(T), V = 16 / es;
    const bool inplace = same(a->xq, a->yq) && (!a->xk.p || same(a->xk, a->yk));
    const bool whole = aligned(a->xq, es) && aligned(a->xk, es) && aligned(a->yq, es) && aligned(a->yk, es) && a->rotary_dim % (a->interleaved ? V : 2 * V) == 0 &&
                       (inplace || (a->head_dim - a->rotary_dim) % V == 0);
    // (chunks of a head that are written; the half layout wants them in one wave)
    const int chunks = (inplace ? a->rotary_dim : a->head_dim) / V;
    const bool vec = whole && (a->interleaved || (chunks <= 64 && (long long)a->batch * a->tokens * (a->heads + a->kv_heads) < (1ll << 31)));
    Params p{};
    auto ten = [](const dpc_seq_tensor& t) { return Ten{(char*)t.p, t.stride_b, t.stride_t, t.stride_h}; };
    p.xq = ten(a->xq); p.xk = ten(a->xk); p.yq = ten(a->yq); p.yk = ten(a->yk);
    p.table = a->table; p.positions = reinterpret_cast<const long long*>(a->positions);
    p.pos_b = a->pos_stride_b; p.start = a->start; p.max_pos = a->max_positions;
    p.total = a->batch * a->tokens; p.heads = a->heads; p.all = a->heads + (a->xk.p ? a->kv_heads : 0);
    p.D = a->head_dim; p.R = a->rotary_dim; p.interleaved = a->interleaved != 0;
    p.rot_items = vec ? p.R / V : p.R / 2;
    const int items = vec ? chunks : p.rot_items + (inplace ? 0 : p.D - p.R);
    // Four heads a thread once the card is full without that (2^20 threads): the angles, the index arithmetic and the position are then shared.
    // Few tokens keep one head a thread, for latency.
    const bool four = (long long)p.total * p.all * items >= (1ll << 20);
    const int groups = four ? (p.all + 3) / 4 : p.all, per_token = groups * items;
    p.tokens = Div(a->tokens); p.items = Div(items); p.per_token = Div(per_token); p.groups = Div(groups);
    p.sign = a->transpose ? -1.f : 1.f;
    constexpr int VV = 16 / (int)sizeof(T);
    if (vec && !a->interleaved) {
        p.per_wg = 64 / items;
        p.work = p.total * groups;
        const dim3 grid((p.work + 4ll * p.per_wg - 1) / (4 * p.per_wg));
        DPC_REQUIRE(grid.x < MAX_GRID, "seq_rotary: grid too large");
        if (four) hipLaunchKernelGGL((rotary_half_kernel<T, 4>), grid, dim3(256), 0, s, p);
        else hipLaunchKernelGGL((rotary_half_kernel<T, 1>), grid, dim3(256), 0, s, p);
        DPC_LAUNCH_CHECK();
        return DPC_OK;
    }
    p.per_wg = std::max(1, 256 / per_token);
    p.work = p.per_wg * per_token;
    const dim3 grid((p.total + (long long)p.per_wg - 1) / p.per_wg, (p.work + 255) / 256);
    DPC_REQUIRE(grid.x < MAX_GRID, "seq_rotary: grid too large");
    if (vec && four) hipLaunchKernelGGL((rotary_kernel<T, VV, 4>), grid, dim3(256), 0, s, p);
    else if (vec) hipLaunchKernelGGL((rotary_kernel<T, VV, 1>), grid, dim3(256), 0, s, p);
    else if (four) hipLaunchKernelGGL((rotary_kernel<T, 1, 4>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((rotary_kernel<T, 1, 1>), grid, dim3(256), 0, s, p);
    DPC_LAUNCH_CHECK();
    return DPC_OK;
}

}  // namespace seqrot
}  // namespace dpc

using namespace dpc;

extern "C" int dpc_seq_rotary_run(const dpc_seq_rotary* a, dpc_stream_t stream) {
    DPC_REQUIRE(a, "seq_rotary: null argument");
    DPC_REQUIRE(a->type >= DPC_SEQ_F32 && a->type <= DPC_SEQ_BF16, "seq_rotary: unknown element type");
    DPC_REQUIRE(a->batch >= 0 && a->tokens >= 0 && a->heads >= 1 && a->head_dim >= 2, "seq_rotary: batch, tokens, heads, head_dim");
    DPC_REQUIRE(a->rotary_dim >= 2 && a->rotary_dim % 2 == 0 && a->rotary_dim <= a->head_dim, "seq_rotary: rotary_dim must be even and at most head_dim");
    DPC_REQUIRE((int64_t)a->batch * a->tokens < (1ll << 31), "seq_rotary: too many tokens");
    if ((int64_t)a->batch * a->tokens == 0) return DPC_OK;
    DPC_REQUIRE(a->xq.p && a->yq.p && a->table && a->max_positions >= 1, "seq_rotary: null argument");
    DPC_REQUIRE(!a->xk.p == !a->yk.p && (!a->xk.p || a->kv_heads >= 1), "seq_rotary: the second tensor needs input, output and heads");
    DPC_REQUIRE((int64_t)(a->heads + a->kv_heads) * a->head_dim < (1 << 23), "seq_rotary: heads x head_dim");
    hipStream_t s = (hipStream_t)stream;
    const int es = a->type == DPC_SEQ_F32 ? 4 : 2;
    ProfScope prof(PROF_SMALL, 0, 2.0 * a->batch * a->tokens * (a->heads + (a->xk.p ? a->kv_heads : 0)) * (double)a->head_dim * es, s);
    return a->type == DPC_SEQ_F32 ? seqrot::run<float>(a, s) : a->type == DPC_SEQ_F16 ? seqrot::run<_Float16>(a, s) : seqrot::run<__bf16>(a, s);
}
