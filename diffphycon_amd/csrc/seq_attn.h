// Attention on token sequences, forward and the backward pass that recomputes the probabilities (include/dpc.h: dpc_seq_attn).
//
//   S = scale Q K^T (masked), lse_i = log sum_j e^S_ij, P = e^(S - lse), O = P V
//   D_i = sum_d dO O,  dV = P^T dO,  dP = dO V^T,  dS = P (dP - D),  dQ = scale dS K,  dK = scale dS^T Q
//
// Every product is a 32 x 32 accumulator tile of one wave.  The tile whose rows are contracted next is computed so that a LANE owns
// the column that survives: in a 32x32 MFMA result lane l holds column l & 31 and the rows rowmap(r, l >> 5).  The forward and the dQ
// kernel compute S^T = K Q^T (column = query), so a query's maximum, sum, lse and D are scalars of a lane pair (l, l ^ 32) and the
// probabilities are already the B operand of O^T += V^T P^T and dQ^T += K^T dS^T; the dK/dV kernel computes S = Q K^T (column = key)
// and its P and dS are the B operands of dV^T += dO^T P and dK^T += Q^T dS.  No probability moves between lanes: the contraction runs
// over the accumulator's own row order, and the other operand is read from LDS in that order (16-bit types: the LDS transpose read).
//
// One source for the three element types: Mma<T> hides the instruction (32x32x16 for 16 bits; for fp32 four 32x32x2, which multiply
// exact fp32) and the operand layouts.  P and dS are rounded to the element type for the second product, as any 16-bit matrix operand
// is; sums and statistics stay fp32.  fp16 has only 2^-14 as its smallest full-precision number: P is carried as 2^15 P and dS under a running power of
// two per column (scale_col), both undone in fp32 at the end.
#pragma once
#include "common.h"

namespace dpc {
namespace seqattn {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int QB = 128;        // rows (queries, or keys in the dK/dV kernel) of a workgroup: 4 waves x 32
constexpr int KB = 64;         // rows of the tile that is staged in LDS

__device__ __forceinline__ int rowmap(int r, int h) { return (r & 3) + 8 * (r >> 2) + 4 * h; }

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((__vector_size__(8)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;

// LDS image of a tile: rows of DP elements in 16-byte chunks.
//  16 bits: pitch DP * 2, chunk c of row r stored at c ^ swz(r): the row read (8 lanes = 8 rows, one chunk) and the transpose read (4
//  rows x 64 bytes) both spread over all banks.  fp32: pitch + 16 bytes does the same for the row read; column reads are contiguous.
template <class T, int DP>
struct Image {
    static constexpr int CH = DP * (int)sizeof(T) / 16;
    static constexpr int PITCH = sizeof(T) == 2 ? DP * 2 : DP * 4 + 16;
    __device__ static __forceinline__ int swz(int r) {
        if (sizeof(T) == 4) return 0;
        return (DP / 32) % 2 ? (r >> 1) & 3 : ((r & 1) << 2) | ((r >> 1) & 3);
    }
    __device__ static __forceinline__ int off(int r, int c) { return r * PITCH + ((c ^ swz(r)) << 4); }
};

template <class T> struct Mma;
template <class T, class F> struct Mma16 {   // the two 16-bit types
    typedef F Frag;
    static constexpr int KS = 16;            // contraction steps of one operand fragment
    template <int DP> __device__ static __forceinline__ Frag row(const char* img, int r, int s, int h) {
        return *reinterpret_cast<const Frag*>(img + Image<T, DP>::off(r, 2 * s + h));
    }
    // fragment of the transposed tile: columns 32 dt .. + 31 as operand rows, contraction over tile rows r0 + 16 s .. in rowmap order
    template <int DP> __device__ static __forceinline__ Frag col(const char* img, int r0, int s, int dt, int lane) {
        const int i = lane & 15, g = (lane >> 4) & 1, h = lane >> 5;
        const int r = 4 * h + (i >> 2);
        const int o = (r0 + 16 * s) * Image<T, DP>::PITCH + Image<T, DP>::off(r, 4 * dt + 2 * g + ((i & 3) >> 1)) + (i & 1) * 8;
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(img + o));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(img + o + 8 * Image<T, DP>::PITCH));
        return __builtin_bit_cast(Frag, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    __device__ static __forceinline__ Frag from_acc(const f32x16& v, int s) {
        f32x8 t;
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = v[8 * s + e];
        return __builtin_convertvector(t, Frag);
    }
};
template <> struct Mma<_Float16> : Mma16<_Float16, f16x8> {
    typedef f16x4 Quad;
    __device__ static __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct Mma<__bf16> : Mma16<__bf16, bf16x8> {
    typedef bf16x4 Quad;
    __device__ static __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mma<float> {
    static constexpr int KS = 8;
    typedef f32x4 Frag;
    typedef f32x4 Quad;
    __device__ static __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
    template <int DP> __device__ static __forceinline__ Frag row(const char* img, int r, int s, int h) {
        return *reinterpret_cast<const Frag*>(img + Image<float, DP>::off(r, 2 * s + h));
    }
    template <int DP> __device__ static __forceinline__ Frag col(const char* img, int r0, int s, int dt, int lane) {
        const int h = lane >> 5;
        Frag f;
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = *reinterpret_cast<const float*>(img + (r0 + 8 * s + 4 * h + e) * Image<float, DP>::PITCH + (32 * dt + (lane & 31)) * 4);
        return f;
    }
    __device__ static __forceinline__ Frag from_acc(const f32x16& v, int s) { return Frag{v[4 * s], v[4 * s + 1], v[4 * s + 2], v[4 * s + 3]}; }
};

struct Ten { char* p; long long b, t, h; };        // strides in bytes

struct Params {
    Ten q, k, v, out, dout, dq, dk, dv;
    float* lse;
    long long lse_b, lse_h;
    const unsigned char* key_mask;
    long long mask_b;
    const int* seqs;
    const int* tiles;                              // [grid / heads][2] or null (dense)
    float *lse2, *delta;                           // backward: lse in powers of two (+inf: a row that sees nothing) and D; lse's addressing
    int heads, kv_heads, group, D, q_len, k_len, causal, tiles_per_seq;
    float scale;
};

struct Seq { long long q0, k0; int ql, kl; };

__device__ __forceinline__ Seq sequence(const Params& p, int b) {
    Seq s;
    if (p.seqs) { s.q0 = p.seqs[4 * b]; s.ql = p.seqs[4 * b + 1]; s.k0 = p.seqs[4 * b + 2]; s.kl = p.seqs[4 * b + 3]; }
    else { s.q0 = 0; s.ql = p.q_len; s.k0 = 0; s.kl = p.k_len; }
    return s;
}

// ROWS x DP tile, global -> registers -> LDS by 256 threads; rows that `ok` refuses and columns >= D become zero.
template <class T, int DP, int ROWS>
struct Stage {
    static constexpr int CH = Image<T, DP>::CH, N = (ROWS * CH + 255) / 256;
    static_assert(ROWS * CH % 256 == 0, "whole rounds");
    uint4 r[N];
    template <class F> __device__ __forceinline__ void issue(const char* base, long long st, int D, F ok) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = threadIdx.x + 256 * i, row = e / CH, c = e % CH;
            r[i] = uint4{0, 0, 0, 0};
            if (c * 16 < D * (int)sizeof(T) && ok(row)) r[i] = *reinterpret_cast<const uint4*>(base + row * st + c * 16);
        }
    }
    __device__ __forceinline__ void store(char* img) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = threadIdx.x + 256 * i, row = e / CH, c = e % CH;
            *reinterpret_cast<uint4*>(img + Image<T, DP>::off(row, c)) = r[i];
        }
    }
};

// operand fragments of one row (this lane's column of the product), zero where !ok
template <class T, int DP>
__device__ __forceinline__ void load_row(typename Mma<T>::Frag (&f)[DP / Mma<T>::KS], const char* row, int h, int D, bool ok) {
#pragma unroll
    for (int s = 0; s < DP / Mma<T>::KS; ++s) {
        uint4 v = {0, 0, 0, 0};
        const int c = 2 * s + h;
        if (ok && c * 16 < D * (int)sizeof(T)) v = *reinterpret_cast<const uint4*>(row + c * 16);
        f[s] = __builtin_bit_cast(typename Mma<T>::Frag, v);
    }
}

// acc[dt] (rows = columns 32 dt .. of the tensor, column = this lane's row) * mul -> row
template <class T, int DP>
__device__ __forceinline__ void store_row(const f32x16 (&acc)[DP / 32], char* row, int h, int D, float mul) {
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * dt + 8 * g + 4 * h;
            if (d < D) {
                const f32x4 v = {acc[dt][4 * g] * mul, acc[dt][4 * g + 1] * mul, acc[dt][4 * g + 2] * mul, acc[dt][4 * g + 3] * mul};
                *reinterpret_cast<typename Mma<T>::Quad*>(row + d * (int)sizeof(T)) = __builtin_convertvector(v, typename Mma<T>::Quad);
            }
        }
}

template <int N> __device__ __forceinline__ void clear(f32x16 (&a)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) a[i][r] = 0.f;
}
template <int N> __device__ __forceinline__ void times(f32x16 (&a)[N], float m) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) a[i][r] *= m;
}

// fp16 only: keep |t| * sc inside fp16 by a power of two per column; when it has to shrink, the column's sum follows.
template <int N> __device__ __forceinline__ void scale_col(f32x16& t, float& sc, f32x16 (&acc)[N]) {
    float m = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) m = fmaxf(m, fabsf(t[r]));
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    if (__any(m * sc > 32768.f)) {
        float ns = sc;
        if (m * sc > 32768.f) ns = ldexpf(1.f, 14 - min(ilogbf(m), 127));
        times(acc, ns / sc);
        sc = ns;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) t[r] *= sc;
}

template <class T> __device__ __forceinline__ constexpr bool is_f16() { return __is_same(T, _Float16); }

// Which keys of the staged tile take part: bit j.  Without a key mask only the sequence's end matters.
__device__ __forceinline__ unsigned long long key_bits(const unsigned char* mask, int kt, int kl, int lane) {
    const int j = kt + lane;
    return __ballot(j < kl && (!mask || mask[j]));
}

template <class T, int DP>
__global__ __launch_bounds__(256) void fwd_kernel(const Params p) {
    typedef Mma<T> M;
    constexpr int NF = DP / M::KS, NP = 32 / M::KS, ND = DP / 32;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    char* const img_k = smem;
    char* const img_v = smem + KB * Image<T, DP>::PITCH;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l31 = lane & 31, h = lane >> 5;
    const int head = blockIdx.x % p.heads, ti = blockIdx.x / p.heads;
    const int b = p.tiles ? p.tiles[2 * ti] : ti / p.tiles_per_seq, tile = p.tiles ? p.tiles[2 * ti + 1] : ti % p.tiles_per_seq;
    const Seq s = sequence(p, b);
    if (tile * QB >= s.ql) return;
    const int kvh = head / p.group, off = s.kl - s.ql;
    const int qw = tile * QB + wave * 32, qi = qw + l31;            // this wave's first query, this lane's
    const bool qok = qi < s.ql;
    const int kend = p.causal ? min(s.kl, min(tile * QB + QB, s.ql) + off) : s.kl;
    const char* const kbase = p.k.p + b * p.k.b + s.k0 * p.k.t + kvh * p.k.h;
    const char* const vbase = p.v.p + b * p.v.b + s.k0 * p.v.t + kvh * p.v.h;
    const unsigned char* const mask = p.key_mask ? p.key_mask + b * p.mask_b + s.k0 : nullptr;
    typename M::Frag qf[NF];
    load_row<T, DP>(qf, p.q.p + b * p.q.b + (s.q0 + (qok ? qi : 0)) * p.q.t + head * p.q.h, h, p.D, qok);
    f32x16 o[ND];
    clear(o);
    // exponents in powers of two; fp16 carries 2^15 P so that small probabilities keep their bits
    const float c = p.scale * LOG2E, lift = is_f16<T>() ? 15.f : 0.f;
    float m = -INFINITY, l = 0.f;                                    // running maximum (scaled), this lane's part of the sum
    Stage<T, DP, KB> sk, sv;
    auto issue = [&](int kt) {
        auto ok = [&](int r) { return kt + r < s.kl && (!mask || mask[kt + r]); };
        sk.issue(kbase + kt * p.k.t, p.k.t, p.D, ok);
        sv.issue(vbase + kt * p.v.t, p.v.t, p.D, ok);
    };
    if (kend > 0) issue(0);
    for (int kt = 0; kt < kend; kt += KB) {
        sk.store(img_k);
        sv.store(img_v);
        __syncthreads();
        if (kt + KB < kend) issue(kt + KB);
        if (!p.causal || kt <= qw + 31 + off) {
            f32x16 st[2];
            clear(st);
#pragma unroll
            for (int sub = 0; sub < 2; ++sub)
#pragma unroll
                for (int f = 0; f < NF; ++f) st[sub] = M::mma(M::template row<DP>(img_k, sub * 32 + l31, f, h), qf[f], st[sub]);
            if (mask || kt + KB > s.kl || (p.causal && kt + KB - 1 > qw + off)) {
                const unsigned long long bits = key_bits(mask, kt, s.kl, lane);
                const int last = p.causal ? qi + off - kt : KB;      // last visible key of the tile
#pragma unroll
                for (int sub = 0; sub < 2; ++sub)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int j = sub * 32 + rowmap(r, h);
                        if (!((bits >> j) & 1) || j > last) st[sub][r] = -INFINITY;
                    }
            }
            float tm = fmaxf(st[0][0], st[1][0]);
#pragma unroll
            for (int r = 1; r < 16; ++r) tm = fmaxf(tm, fmaxf(st[0][r], st[1][r]));
            tm = fmaxf(tm, __shfl_xor(tm, 32, 64));
            const float mn = fmaxf(m, tm * c);
            const float sub0 = (mn == -INFINITY ? 0.f : mn) - lift;
            const float alpha = exp2f(m - (mn == -INFINITY ? 0.f : mn));
            m = mn;
            float sum = 0.f;
#pragma unroll
            for (int sub = 0; sub < 2; ++sub)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    st[sub][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[sub][r], c, -sub0));
                    sum += st[sub][r];
                }
            l = l * alpha + sum;
            times(o, alpha);
#pragma unroll
            for (int sub = 0; sub < 2; ++sub)
#pragma unroll
                for (int f = 0; f < NP; ++f) {
                    const typename M::Frag pf = M::from_acc(st[sub], f);
#pragma unroll
                    for (int dt = 0; dt < ND; ++dt) o[dt] = M::mma(M::template col<DP>(img_v, sub * 32, f, dt, lane), pf, o[dt]);
                }
        }
        __syncthreads();
    }
    l += __shfl_xor(l, 32, 64);
    if (!qok) return;
    store_row<T, DP>(o, p.out.p + b * p.out.b + (s.q0 + qi) * p.out.t + head * p.out.h, h, p.D, l == 0.f ? 0.f : 1.f / l);
    if (h == 0) p.lse[b * p.lse_b + head * p.lse_h + s.q0 + qi] = l == 0.f ? -INFINITY : (m - lift + log2f(l)) * LN2;
}

// lse2 = lse in powers of two (+inf where the row saw nothing: e^(S - inf) = 0), delta = sum_d dO O; 16 lanes a row
template <class T>
__global__ __launch_bounds__(256) void delta_kernel(const Params p) {
    const int head = blockIdx.x % p.heads, ti = blockIdx.x / p.heads;
    const int b = p.tiles ? p.tiles[2 * ti] : ti / p.tiles_per_seq, tile = p.tiles ? p.tiles[2 * ti + 1] : ti % p.tiles_per_seq;
    const Seq s = sequence(p, b);
    constexpr int E = 16 / (int)sizeof(T);
    typedef T V __attribute__((ext_vector_type(E)));
    const int part = threadIdx.x & 15;
    for (int r = threadIdx.x >> 4; r < QB; r += 16) {
        const int i = tile * QB + r;
        if (i >= s.ql) break;
        const char* o = p.out.p + b * p.out.b + (s.q0 + i) * p.out.t + head * p.out.h;
        const char* g = p.dout.p + b * p.dout.b + (s.q0 + i) * p.dout.t + head * p.dout.h;
        float acc = 0.f;
        for (int c = part; c * E < p.D; c += 16) {
            const V a = *reinterpret_cast<const V*>(o + c * 16), e = *reinterpret_cast<const V*>(g + c * 16);
#pragma unroll
            for (int k = 0; k < E; ++k) acc = __builtin_fmaf((float)a[k], (float)e[k], acc);
        }
#pragma unroll
        for (int x = 8; x; x >>= 1) acc += __shfl_xor(acc, x, 64);
        if (part == 0) {
            const long long at = b * p.lse_b + head * p.lse_h + s.q0 + i;
            const float v = p.lse[at];
            p.lse2[at] = v == -INFINITY ? INFINITY : v * LOG2E;
            p.delta[at] = v == -INFINITY ? 0.f : acc;
        }
    }
}

template <class T, int DP>
__global__ __launch_bounds__(256) void dq_kernel(const Params p) {
    typedef Mma<T> M;
    constexpr int NF = DP / M::KS, NP = 32 / M::KS, ND = DP / 32;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    char* const img_k = smem;
    char* const img_v = smem + KB * Image<T, DP>::PITCH;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l31 = lane & 31, h = lane >> 5;
    const int head = blockIdx.x % p.heads, ti = blockIdx.x / p.heads;
    const int b = p.tiles ? p.tiles[2 * ti] : ti / p.tiles_per_seq, tile = p.tiles ? p.tiles[2 * ti + 1] : ti % p.tiles_per_seq;
    const Seq s = sequence(p, b);
    if (tile * QB >= s.ql) return;
    const int kvh = head / p.group, off = s.kl - s.ql;
    const int qw = tile * QB + wave * 32, qi = qw + l31;
    const bool in = qi < s.ql;
    const int kend = p.causal ? min(s.kl, min(tile * QB + QB, s.ql) + off) : s.kl;
    const char* const kbase = p.k.p + b * p.k.b + s.k0 * p.k.t + kvh * p.k.h;
    const char* const vbase = p.v.p + b * p.v.b + s.k0 * p.v.t + kvh * p.v.h;
    const unsigned char* const mask = p.key_mask ? p.key_mask + b * p.mask_b + s.k0 : nullptr;
    const long long at = b * p.lse_b + head * p.lse_h + s.q0 + (in ? qi : 0);
    const float lse2 = in ? p.lse2[at] : INFINITY, delta = in ? p.delta[at] : 0.f;
    const bool sees = lse2 != INFINITY;                              // (a row that sees nothing takes no part, whatever it holds)
    typename M::Frag qf[NF], gf[NF];
    const long long row = s.q0 + (in ? qi : 0);
    load_row<T, DP>(qf, p.q.p + b * p.q.b + row * p.q.t + head * p.q.h, h, p.D, sees);
    load_row<T, DP>(gf, p.dout.p + b * p.dout.b + row * p.dout.t + head * p.dout.h, h, p.D, sees);
    f32x16 acc[ND];
    clear(acc);
    const float c = p.scale * LOG2E;
    float sc = is_f16<T>() ? 0x1p100f : 1.f;
    Stage<T, DP, KB> sk, sv;
    auto issue = [&](int kt) {
        auto ok = [&](int r) { return kt + r < s.kl && (!mask || mask[kt + r]); };
        sk.issue(kbase + kt * p.k.t, p.k.t, p.D, ok);
        sv.issue(vbase + kt * p.v.t, p.v.t, p.D, ok);
    };
    if (kend > 0) issue(0);
    for (int kt = 0; kt < kend; kt += KB) {
        sk.store(img_k);
        sv.store(img_v);
        __syncthreads();
        if (kt + KB < kend) issue(kt + KB);
        if (!p.causal || kt <= qw + 31 + off) {
            const bool partial = mask || kt + KB > s.kl || (p.causal && kt + KB - 1 > qw + off);
            const unsigned long long bits = partial ? key_bits(mask, kt, s.kl, lane) : ~0ull;
            const int last = p.causal ? qi + off - kt : KB;
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
                f32x16 st[1], dp[1];
                clear(st);
                clear(dp);
#pragma unroll
                for (int f = 0; f < NF; ++f) st[0] = M::mma(M::template row<DP>(img_k, sub * 32 + l31, f, h), qf[f], st[0]);
#pragma unroll
                for (int f = 0; f < NF; ++f) dp[0] = M::mma(M::template row<DP>(img_v, sub * 32 + l31, f, h), gf[f], dp[0]);
#pragma unroll
                for (int r = 0; r < 16; ++r) st[0][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[0][r], c, -lse2)) * (dp[0][r] - delta);
                if (partial) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int j = sub * 32 + rowmap(r, h);
                        if (!((bits >> j) & 1) || j > last) st[0][r] = 0.f;
                    }
                }
                if (is_f16<T>()) scale_col(st[0], sc, acc);
#pragma unroll
                for (int f = 0; f < NP; ++f) {
                    const typename M::Frag df = M::from_acc(st[0], f);
#pragma unroll
                    for (int dt = 0; dt < ND; ++dt) acc[dt] = M::mma(M::template col<DP>(img_k, sub * 32, f, dt, lane), df, acc[dt]);
                }
            }
        }
        __syncthreads();
    }
    if (in) store_row<T, DP>(acc, p.dq.p + b * p.dq.b + row * p.dq.t + head * p.dq.h, h, p.D, p.scale / sc);
}

template <class T, int DP>
__global__ __launch_bounds__(256) void dkv_kernel(const Params p) {
    typedef Mma<T> M;
    constexpr int NF = DP / M::KS, NP = 32 / M::KS, ND = DP / 32;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    char* const img_q = smem;
    char* const img_g = smem + KB * Image<T, DP>::PITCH;
    float* const s_lse = reinterpret_cast<float*>(smem + 2 * KB * Image<T, DP>::PITCH);     // [64] lse2, [64] delta
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l31 = lane & 31, h = lane >> 5;
    const int kvh = blockIdx.x % p.kv_heads, ti = blockIdx.x / p.kv_heads;
    const int b = p.tiles ? p.tiles[2 * ti] : ti / p.tiles_per_seq, tile = p.tiles ? p.tiles[2 * ti + 1] : ti % p.tiles_per_seq;
    const Seq s = sequence(p, b);
    if (tile * QB >= s.kl) return;
    const int off = s.kl - s.ql;
    const int kw = tile * QB + wave * 32, kj = kw + l31;             // this wave's first key, this lane's
    const bool in = kj < s.kl;
    const long long row = s.k0 + (in ? kj : 0);
    const bool live = in && (!p.key_mask || p.key_mask[b * p.mask_b + row]);
    typename M::Frag kf[NF], vf[NF];
    load_row<T, DP>(kf, p.k.p + b * p.k.b + row * p.k.t + kvh * p.k.h, h, p.D, live);
    load_row<T, DP>(vf, p.v.p + b * p.v.b + row * p.v.t + kvh * p.v.h, h, p.D, live);
    f32x16 dk[ND], dv[ND];
    clear(dk);
    clear(dv);
    const float c = p.scale * LOG2E, lift = is_f16<T>() ? 15.f : 0.f;
    float sc = is_f16<T>() ? 0x1p100f : 1.f;
    const int qbegin = p.causal ? max(0, tile * QB - off) / KB * KB : 0;        // first tile with a query that sees the first key
    const int per_head = qbegin < s.ql ? (s.ql - qbegin + KB - 1) / KB : 0, steps = per_head * p.group;
    Stage<T, DP, KB> sq, sg;
    float r_lse = INFINITY, r_delta = 0.f;
    auto issue = [&](int step) {
        const int head = kvh * p.group + step / per_head, qt = qbegin + step % per_head * KB;
        const long long first = s.q0 + qt, at = b * p.lse_b + head * p.lse_h + first;
        const float* const lse2 = p.lse2 + at;
        auto ok = [&](int r) { return qt + r < s.ql && lse2[r] != INFINITY; };
        sq.issue(p.q.p + b * p.q.b + first * p.q.t + head * p.q.h, p.q.t, p.D, ok);
        sg.issue(p.dout.p + b * p.dout.b + first * p.dout.t + head * p.dout.h, p.dout.t, p.D, ok);
        if (tid < KB) {
            r_lse = qt + tid < s.ql ? lse2[tid] : INFINITY;
            r_delta = qt + tid < s.ql ? p.delta[at + tid] : 0.f;
        }
    };
    if (steps > 0) issue(0);
    for (int step = 0; step < steps; ++step) {
        const int qt = qbegin + step % per_head * KB;
        sq.store(img_q);
        sg.store(img_g);
        if (tid < KB) { s_lse[tid] = r_lse - lift; s_lse[KB + tid] = r_delta; }
        __syncthreads();
        if (step + 1 < steps) issue(step + 1);
        if (!p.causal || qt + KB - 1 >= kw - off) {
            const bool partial = p.causal && kw + 31 - off > qt;
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
                f32x16 st[1], dp[1];
                clear(st);
                clear(dp);
#pragma unroll
                for (int f = 0; f < NF; ++f) st[0] = M::mma(M::template row<DP>(img_q, sub * 32 + l31, f, h), kf[f], st[0]);
#pragma unroll
                for (int f = 0; f < NF; ++f) dp[0] = M::mma(M::template row<DP>(img_g, sub * 32 + l31, f, h), vf[f], dp[0]);
                const float* const sl = s_lse + sub * 32 + 4 * h;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4 le = *reinterpret_cast<const f32x4*>(sl + 8 * g), de = *reinterpret_cast<const f32x4*>(sl + KB + 8 * g);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = 4 * g + e;
                        float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(st[0][r], c, -le[e]));
                        if (partial && kj - off > qt + sub * 32 + rowmap(r, h)) pr = 0.f;
                        st[0][r] = pr;
                        dp[0][r] = pr * (dp[0][r] - de[e]);
                    }
                }
                if (is_f16<T>()) scale_col(dp[0], sc, dk);
#pragma unroll
                for (int f = 0; f < NP; ++f) {
                    const typename M::Frag pf = M::from_acc(st[0], f), df = M::from_acc(dp[0], f);
#pragma unroll
                    for (int dt = 0; dt < ND; ++dt) dv[dt] = M::mma(M::template col<DP>(img_g, sub * 32, f, dt, lane), pf, dv[dt]);
#pragma unroll
                    for (int dt = 0; dt < ND; ++dt) dk[dt] = M::mma(M::template col<DP>(img_q, sub * 32, f, dt, lane), df, dk[dt]);
                }
            }
        }
        __syncthreads();
    }
    if (!in) return;
    if (!live) { clear(dk); clear(dv); }
    const float un = is_f16<T>() ? 0x1p-15f : 1.f;                   // (P and with it dS carry 2^15)
    store_row<T, DP>(dk, p.dk.p + b * p.dk.b + row * p.dk.t + kvh * p.dk.h, h, p.D, p.scale * un / sc);
    store_row<T, DP>(dv, p.dv.p + b * p.dv.b + row * p.dv.t + kvh * p.dv.h, h, p.D, un);
}

template <class T, int DP>
int run_fwd(const Params& p, int grid, hipStream_t s) {
    constexpr int lds = 2 * KB * Image<T, DP>::PITCH;
    static DeviceOnce once;
    if (!once) { DPC_HIP(hipFuncSetAttribute((const void*)fwd_kernel<T, DP>, hipFuncAttributeMaxDynamicSharedMemorySize, lds)); once = true; }
    hipLaunchKernelGGL((fwd_kernel<T, DP>), dim3(grid), dim3(256), lds, s, p);
    DPC_LAUNCH_CHECK();
    return DPC_OK;
}

template <class T, int DP>
int run_bwd(const Params& pq, int grid_q, const Params& pk, int grid_k, hipStream_t s) {
    constexpr int lds = 2 * KB * Image<T, DP>::PITCH, lds_k = lds + 2 * KB * 4;
    static DeviceOnce once;
    if (!once) {
        DPC_HIP(hipFuncSetAttribute((const void*)dq_kernel<T, DP>, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
        DPC_HIP(hipFuncSetAttribute((const void*)dkv_kernel<T, DP>, hipFuncAttributeMaxDynamicSharedMemorySize, lds_k));
        once = true;
    }
    if (grid_q) {
        hipLaunchKernelGGL((delta_kernel<T>), dim3(grid_q), dim3(256), 0, s, pq);
        DPC_LAUNCH_CHECK();
        hipLaunchKernelGGL((dq_kernel<T, DP>), dim3(grid_q), dim3(256), lds, s, pq);
        DPC_LAUNCH_CHECK();
    }
    if (grid_k) {
        hipLaunchKernelGGL((dkv_kernel<T, DP>), dim3(grid_k), dim3(256), lds_k, s, pk);
        DPC_LAUNCH_CHECK();
    }
    return DPC_OK;
}

// one element type's kernels live in one translation unit (seq_attn_{f32,f16,bf16}.hip)
template <class T> int fwd(const Params& p, int grid, hipStream_t s) {
    return p.D <= 32 ? run_fwd<T, 32>(p, grid, s) : p.D <= 64 ? run_fwd<T, 64>(p, grid, s) : p.D <= 96 ? run_fwd<T, 96>(p, grid, s) : run_fwd<T, 128>(p, grid, s);
}
template <class T> int bwd(const Params& pq, int gq, const Params& pk, int gk, hipStream_t s) {
    return pq.D <= 32 ? run_bwd<T, 32>(pq, gq, pk, gk, s) : pq.D <= 64 ? run_bwd<T, 64>(pq, gq, pk, gk, s)
         : pq.D <= 96 ? run_bwd<T, 96>(pq, gq, pk, gk, s) : run_bwd<T, 128>(pq, gq, pk, gk, s);
}
int fwd_f32(const Params&, int, hipStream_t);
int fwd_f16(const Params&, int, hipStream_t);
int fwd_bf16(const Params&, int, hipStream_t);
int bwd_f32(const Params&, int, const Params&, int, hipStream_t);
int bwd_f16(const Params&, int, const Params&, int, hipStream_t);
int bwd_bf16(const Params&, int, const Params&, int, hipStream_t);

}  // namespace seqattn
}  // namespace dpc
