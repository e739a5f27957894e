// Rotary positions (include/dpc.h: dpc_seq_rotary): pair (a, b) of a head at position p becomes (a cos t - b sin t, a sin t + b cos t)
// with (cos, sin) = table[p][pair]; the gradient is the transpose (sin -> -sin), so both directions are this kernel.
// Bound by bytes: every element is read and written once.  A thread owns one chunk of a token's head -- 16 bytes of pairs (interleaved),
// 16 bytes of each half (half layout), or 16 bytes of the pass-through part -- and walks over heads with the chunk's cosines in registers.
// Rows that do not start on 16 bytes, or halves that do not, go one pair at a time.
#include <algorithm>

#include "common.h"

namespace dpc {
namespace seqrot {

struct Ten { char* p; long long b, t, h; };      // strides in elements
struct Params {
    Ten xq, xk, yq, yk;
    const float* table;
    const long long* positions;
    long long pos_b, start, max_pos;
    int tokens, total, heads, kv_heads, D, R, interleaved, items, rot_items, hgroups, per_wg;
    float sign;
};

template <class T, int V>        // V: elements of an access (16 bytes, or 1)
__global__ __launch_bounds__(256) void rotary_kernel(const Params p) {
    typedef T Q __attribute__((ext_vector_type(V)));
    constexpr int P = V > 1 ? V : 2;                                 // elements a chunk may hold per side
    const int per_token = p.hgroups * p.items;
    for (int w = threadIdx.x; w < p.per_wg * per_token; w += 256) {
        const int lt = w / per_token, in = w % per_token, hg = in / p.items, it = in % p.items;
        const long long n = (long long)blockIdx.x * p.per_wg + lt;
        if (n >= p.total) return;
        const int b = (int)n / p.tokens, t = (int)n % p.tokens;
        const bool turn = it < p.rot_items;
        // first element of the chunk, distance to the pair's other side (half layout), pairs in it
        int c0, other = 0, i0 = 0;
        if (!turn) c0 = p.R + (it - p.rot_items) * V;
        else if (p.interleaved) { c0 = it * P; i0 = it * (P / 2); }
        else { c0 = it * V; other = p.R / 2; i0 = it * V; }
        constexpr int NP = V > 1 ? V : 1;                            // pairs held at most (half layout: V, interleaved: V / 2)
        float cs[NP], sn[NP];
        if (turn) {
            const long long pos = p.positions ? p.positions[b * p.pos_b + t] : p.start + t;
            const bool ok = pos >= 0 && pos < p.max_pos;
            const float2* tab = reinterpret_cast<const float2*>(p.table) + (ok ? pos : 0) * (p.R / 2) + i0;
            const int np = p.interleaved ? P / 2 : NP;
#pragma unroll
            for (int k = 0; k < NP; ++k)
                if (k < np) {
                    const float2 z = tab[k];
                    cs[k] = ok ? z.x : __builtin_nanf("");
                    sn[k] = ok ? z.y * p.sign : __builtin_nanf("");
                }
        }
        for (int hd = hg; hd < p.heads + p.kv_heads; hd += p.hgroups) {
            const bool isq = hd < p.heads;
            const Ten& X = isq ? p.xq : p.xk;
            const Ten& Y = isq ? p.yq : p.yk;
            const int h = isq ? hd : hd - p.heads;
            const T* x = reinterpret_cast<const T*>(X.p) + b * X.b + t * X.t + h * X.h + c0;
            T* y = reinterpret_cast<T*>(Y.p) + b * Y.b + t * Y.t + h * Y.h + c0;
            if (!turn) {
                *reinterpret_cast<Q*>(y) = *reinterpret_cast<const Q*>(x);
            } else if (p.interleaved) {
                if constexpr (V > 1) {
                    Q q = *reinterpret_cast<const Q*>(x);
#pragma unroll
                    for (int k = 0; k < V / 2; ++k) {
                        const float a = (float)q[2 * k], c = (float)q[2 * k + 1];
                        q[2 * k] = (T)(a * cs[k] - c * sn[k]);
                        q[2 * k + 1] = (T)(a * sn[k] + c * cs[k]);
                    }
                    *reinterpret_cast<Q*>(y) = q;
                } else {
                    const float a = (float)x[0], c = (float)x[1];
                    y[0] = (T)(a * cs[0] - c * sn[0]);
                    y[1] = (T)(a * sn[0] + c * cs[0]);
                }
            } else {
                Q q = *reinterpret_cast<const Q*>(x), u = *reinterpret_cast<const Q*>(x + other);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const float a = (float)q[k], c = (float)u[k];
                    q[k] = (T)(a * cs[k] - c * sn[k]);
                    u[k] = (T)(a * sn[k] + c * cs[k]);
                }
                *reinterpret_cast<Q*>(y) = q;
                *reinterpret_cast<Q*>(y + other) = u;
            }
        }
    }
}

static bool aligned(const dpc_seq_tensor& t, int es) {
    return !t.p || ((size_t)t.p | (size_t)(t.stride_b * es) | (size_t)(t.stride_t * es) | (size_t)(t.stride_h * es)) % 16 == 0;
}

static bool same(const dpc_seq_tensor& a, const dpc_seq_tensor& b) {
    return a.p == b.p && a.stride_b == b.stride_b && a.stride_t == b.stride_t && a.stride_h == b.stride_h;
}

template <class T> int run(const dpc_seq_rotary* a, hipStream_t s) {
    const int es = (int)sizeof(T), V = 16 / es;
    const bool inplace = same(a->xq, a->yq) && (!a->xk.p || same(a->xk, a->yk));
    const bool vec = aligned(a->xq, es) && aligned(a->xk, es) && aligned(a->yq, es) && aligned(a->yk, es) && a->rotary_dim % (a->interleaved ? V : 2 * V) == 0 &&
                     (inplace || (a->head_dim - a->rotary_dim) % V == 0);
    Params p{};
    auto ten = [](const dpc_seq_tensor& t) { return Ten{(char*)t.p, t.stride_b, t.stride_t, t.stride_h}; };
    p.xq = ten(a->xq); p.xk = ten(a->xk); p.yq = ten(a->yq); p.yk = ten(a->yk);
    p.table = a->table; p.positions = reinterpret_cast<const long long*>(a->positions);
    p.pos_b = a->pos_stride_b; p.start = a->start; p.max_pos = a->max_positions;
    p.tokens = a->tokens; p.total = a->batch * a->tokens; p.heads = a->heads; p.kv_heads = a->xk.p ? a->kv_heads : 0;
    p.D = a->head_dim; p.R = a->rotary_dim; p.interleaved = a->interleaved != 0;
    const int w = vec ? V : 1;
    p.rot_items = p.interleaved ? p.R / (vec ? V : 2) : p.R / 2 / w;
    p.items = p.rot_items + (inplace ? 0 : (p.D - p.R) / w);
    const int all = p.heads + p.kv_heads;
    p.hgroups = all;
    p.per_wg = std::max(1, 256 / (p.hgroups * p.items));
    p.sign = a->transpose ? -1.f : 1.f;
    const int grid = (p.total + p.per_wg - 1) / p.per_wg;
    if (vec) hipLaunchKernelGGL((rotary_kernel<T, 16 / (int)sizeof(T)>), dim3(grid), dim3(256), 0, s, p);
    else hipLaunchKernelGGL((rotary_kernel<T, 1>), dim3(grid), dim3(256), 0, s, p);
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
    DPC_REQUIRE((int64_t)(a->heads + a->kv_heads) * a->head_dim < (1 << 24), "seq_rotary: heads x head_dim");
    hipStream_t s = (hipStream_t)stream;
    const int es = a->type == DPC_SEQ_F32 ? 4 : 2;
    ProfScope prof(PROF_SMALL, 0, 2.0 * a->batch * a->tokens * (a->heads + (a->xk.p ? a->kv_heads : 0)) * (double)a->head_dim * es, s);
    return a->type == DPC_SEQ_F32 ? seqrot::run<float>(a, s) : a->type == DPC_SEQ_F16 ? seqrot::run<_Float16>(a, s) : seqrot::run<__bf16>(a, s);
}
