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
// One source for the three element types.  Mma<T> hides the 16-bit instruction (32x32x16) and the operand layouts; fp32 goes through the same
// instruction as three bf16 parts (Split3), but for few rows, where the native fp32 one is used.  P and dS are rounded to the element type for the
// second product, as any 16-bit matrix operand is; sums and statistics stay fp32.  fp16 has only 2^-14 as its smallest full-precision number: P is
// carried as 2^7 P (forward) or 2^15 P and dS under a running power of two per column (shrink_col), both undone in fp32 at the end.
//
// What bounds it (counters at the sizes named at the kernels; figures of one card, on which a large library product reaches 1248 TFLOP/s in bf16, 1184 in fp16 and
// 154 in fp32): in 16 bits the matrix and the vector units take turns, and neither is a bound yet.  Head size 128: busy 0.47 and 0.46 of the time in the
// forward (900 TFLOP/s executed), 0.50 and 0.43 in dQ (915), 0.44 and 0.38 in dK/dV (875); head size 64, with more exponentials, maxima and masks for a
// product: 0.33 and 0.64 (575), 0.30 and 0.67 (535), 0.27 and 0.53 (500).  fp32, six bf16 products for one, overlaps them
// better: 0.53 to 0.63 and, for the vector units split operands, 0.62 to 0.71 (165 to 185 of fp32's products).
// The backward pass executes seven products where five would do, for dQ and dK/dV are summed by different workgroups and nothing is added with atomics.
#pragma once
#include <algorithm>
#include <type_traits>

#include "bf16x6.h"
#include "seq_div.h"

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

// LDS image of a tile: rows of DP elements in 16-byte chunks, filled 16 bytes a lane straight from global memory (Stage), so the image
// has no padding; chunk c of row r is stored at c ^ swz(r).  LDS serves a 16-byte read 16 lanes at a time over 64 banks (256 bytes): the row read
// (lane = row, one chunk) wants 16 rows in 16 different 16-byte slots, the transpose read (4 rows x 64 bytes) 4 rows in 4 different
// 64-byte ones.  With rows of 256 bytes all of that has to come from swz, with shorter ones a part comes from where the row starts.
template <class T, int DP>
struct Image {
    static constexpr int CH = DP * (int)sizeof(T) / 16, PITCH = CH * 16;
    __device__ static __forceinline__ int swz(int r) {
        return CH % 16 == 0 ? ((r & 3) << 2) | ((r >> 2) & 3) : CH % 8 == 0 ? ((r & 2) << 1) | ((r >> 2) & 3) : (r >> 2) & 3;
    }
    __device__ static __forceinline__ int off(int r, int c) { return r * PITCH + ((c ^ swz(r)) << 4); }
};

template <class T> struct Mma;
template <class T, class F> struct Mma16 {   // the two 16-bit types
    typedef F Frag;
    static constexpr int KS = 16;            // contraction steps of one operand fragment
    template <int DP, int PLANE = 0> __device__ static __forceinline__ Frag row(const char* img, int r, int s, int h) {
        return *reinterpret_cast<const Frag*>(img + Image<T, DP>::off(r, 2 * s + h));
    }
    // fragment of the transposed tile: columns 32 dt .. + 31 as operand rows, contraction over tile rows r0 + 16 s .. in rowmap order
    template <int DP, int PLANE = 0> __device__ static __forceinline__ Frag col(const char* img, int r0, int s, int dt, int lane) {
        const int i = lane & 15, g = (lane >> 4) & 1, h = lane >> 5;
        const int r = 4 * h + (i >> 2);
        const int c = 4 * dt + 2 * g + ((i & 3) >> 1), o = (r0 + 16 * s) * Image<T, DP>::PITCH + (i & 1) * 8;       // (swz repeats every 16 rows)
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(img + o + Image<T, DP>::off(r, c)));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(img + o + Image<T, DP>::off(r + 8, c)));
        return __builtin_bit_cast(Frag, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    __device__ static __forceinline__ float value(const Frag& f, int e) { return (float)f[e]; }
    __device__ static __forceinline__ Frag from_acc(const f32x16& v, int s) {
        f32x8 t;
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = v[8 * s + e];
        return __builtin_convertvector(t, Frag);
    }
    __device__ static __forceinline__ Frag rest(const f32x16& v, int s, const Frag& f) {          // what from_acc's rounding left
        f32x8 t;
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = v[8 * s + e] - (float)f[e];
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
    template <int DP, int PLANE = 0> __device__ static __forceinline__ Frag row(const char* img, int r, int s, int h) {
        return *reinterpret_cast<const Frag*>(img + Image<float, DP>::off(r, 2 * s + h));
    }
    template <int DP, int PLANE = 0> __device__ static __forceinline__ Frag col(const char* img, int r0, int s, int dt, int lane) {
        const int h = lane >> 5;
        Frag f;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            f[e] = *reinterpret_cast<const float*>(img + Image<float, DP>::off(r0 + 8 * s + 4 * h + e, 8 * dt + ((lane & 31) >> 2)) + (lane & 3) * 4);
        return f;
    }
    __device__ static __forceinline__ float value(const Frag& f, int e) { return f[e]; }
    __device__ static __forceinline__ Frag from_acc(const f32x16& v, int s) { return Frag{v[4 * s], v[4 * s + 1], v[4 * s + 2], v[4 * s + 3]}; }
};

// fp32 by the bf16 matrix instructions: x = x1 + x2 + x3 in three bf16 parts, exactly (bf16x6.h), and six of the nine products -- what is left out is
// below 2^-24 of |a b|, an fp32 product's own rounding.  6 / 16 of the native instruction's time (1 x 4096, 16 heads of 128: the forward takes
// 0.6 of the time that it took with those).  An operand is three fragments, an image three 16-bit images PLANE bytes apart.
struct Split3 {
    typedef struct { bf16x8 p[3]; } Frag;
    typedef f32x4 Quad;
    typedef Mma<__bf16> B;
    static constexpr int KS = 16;
    __device__ static __forceinline__ f32x16 mma(const Frag& a, const Frag& b, f32x16 c) {
        b6::mfma6(c, a.p, b.p);
        return c;
    }
    template <int DP, int PLANE> __device__ static __forceinline__ Frag row(const char* img, int r, int s, int h) {
        return Frag{{B::row<DP>(img, r, s, h), B::row<DP>(img + PLANE, r, s, h), B::row<DP>(img + 2 * PLANE, r, s, h)}};
    }
    template <int DP, int PLANE> __device__ static __forceinline__ Frag col(const char* img, int r0, int s, int dt, int lane) {
        return Frag{{B::col<DP>(img, r0, s, dt, lane), B::col<DP>(img + PLANE, r0, s, dt, lane), B::col<DP>(img + 2 * PLANE, r0, s, dt, lane)}};
    }
    __device__ static __forceinline__ float value(const Frag& f, int e) { return (float)f.p[0][e] + ((float)f.p[1][e] + (float)f.p[2][e]); }
    __device__ static __forceinline__ Frag of(const float (&v)[8]) {
        Frag f;
        b6::split8(v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], f.p);
        return f;
    }
    __device__ static __forceinline__ Frag from_acc(const f32x16& v, int s) {
        const float t[8] = {v[8 * s], v[8 * s + 1], v[8 * s + 2], v[8 * s + 3], v[8 * s + 4], v[8 * s + 5], v[8 * s + 6], v[8 * s + 7]};
        return of(t);
    }
};
template <class T> constexpr bool SPLIT = sizeof(T) == 4;
template <class T> using Op = std::conditional_t<SPLIT<T>, Split3, Mma<T>>;

struct Ten { char* p; long long b, t, h; };        // strides in bytes

struct Params {
    Ten q, k, v, out, dout, dq, dk, dv;
    float* lse;
    long long lse_b, lse_h;                        // row numbers of q, as in lse
    const unsigned char* key_mask;
    long long mask_b;
    const int* tiles;                              // [..][8] = (sequence, block, first query, queries, first key, keys, ..) or null (dense)
    float *lse2, *ndelta;                          // backward: lse in powers of two (+inf: a row that sees nothing) and -D, numbered like lse
    // splits: partial sums [split][row][D] and per-row scalars (layout at each kernel).  Rows are numbered block by block, not as they lie in the
    // tensors: scratch goes by the blocks that there are, and a plan of short sequences in a long buffer has few.
    float *part, *part_ml;
    long long part_rows;
    int block_rows;                                // most rows that a block has
    int heads, kv_heads, group, D, q_len, k_len, causal, n_tiles, tiles_per_seq, band_tiles, pairs, splits, few;
    // splits, sub-blocks of a block, kv_heads, group, pairs; workgroups of a pair in a band of blocks and in the last band, of a band on an XCD
    Div by_split, by_sub, by_kv, by_group, by_tile, by_pair, by_last, by_band;
    float scale;
};

// Which block of which (sequence, key head) a workgroup has.  Workgroups go round the 8 XCDs, each with its own L2: the blocks of one
// (sequence, key head), which read the same keys and values, stay on one XCD where the pairs divide evenly, and follow each other.  Under a causal mask
// they differ in work (the last queries', the first keys' have most): then the quarter with most work of every pair comes first, so that
// none of it is left for the end (pair after pair: 20 to 40 % of the card idle at the end; all pairs' heaviest blocks first: keys and values leave L2
// in between).  A query block is `subs` sub-blocks of QB rows (rows = tokens x heads of the group).
struct Where {
    int b, tile, kvh, sub, split, ql, kl, block;                     // block: which of all blocks, of (sequence, key head) too
    long long q0, k0;
    __device__ __forceinline__ long long part(const Params& p, int row) const { return (long long)block * p.block_rows + row; }
};
__device__ __forceinline__ Where where(const Params& p, bool last_first) {
    Where w;
    int id = blockIdx.x;
    w.ql = p.q_len; w.kl = p.k_len; w.q0 = w.k0 = 0;
    if (p.tiles) {
        w.split = p.by_split.take(id);
        w.block = id;
        w.sub = p.by_sub.take(id);
        w.kvh = p.by_kv.take(id);
        const int* e = p.tiles + 8 * (long long)id;
        w.b = e[0]; w.tile = e[1]; w.q0 = e[2]; w.ql = e[3]; w.k0 = e[4]; w.kl = e[5];
        return w;
    }
    int pair, i;
    if (p.pairs % 8 == 0) {
        int band = id >> 3;
        pair = p.by_band.take(band);                                 // place within the band
        i = ((band + 1) * p.band_tiles < p.tiles_per_seq ? p.by_pair : p.by_last).take(pair) + band * (int)p.by_pair.d;
        pair += (id & 7) * (p.pairs >> 3);
    } else {
        i = id;
        pair = p.by_tile.take(i);
    }
    w.split = p.by_split.take(i);
    w.block = pair * p.tiles_per_seq * (int)p.by_sub.d + i;
    w.sub = p.by_sub.take(i);
    w.tile = last_first ? p.tiles_per_seq - 1 - i : i;
    w.kvh = p.by_kv.take(pair);
    w.b = pair;
    return w;
}

// Sources of 16 (4) bytes for rows and columns that are not there: zeros, and +inf for their lse
__device__ __attribute__((aligned(16))) const float FILL[8] = {0.f, 0.f, 0.f, 0.f, INFINITY, 0.f, 0.f, 0.f};

// Copies 16 (4) bytes a lane from global memory to LDS at `lds` + 16 (4) * lane, past the registers.  Written out, because the compiler would wait for
// every such copy in flight before any LDS read; copies_done() is the wait, followed by a barrier.  (A write to m0 needs one wait state before its use.)
__device__ __forceinline__ void copy16(const char* src, unsigned lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" :: "v"(src), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void copy16(const char* base, unsigned off, unsigned lds) {          // one base for the wave
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" :: "v"(off), "s"(base), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void copy4(const char* src, unsigned lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" :: "v"(src), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void copies_done() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ unsigned lds_offset(const void* p) {
    return __builtin_amdgcn_readfirstlane((unsigned)(size_t)(__attribute__((address_space(3))) const char*)p);
}

// Bits of 64 rows, tested by 32-bit shifts alone: a 64-bit shift whose amount is the last vector register that a wave has reads register 0 instead
// when the wave's registers end the register file (seen in the fp32 kernel of 256 registers: masked keys counted; the build refuses such a shift).
__device__ __forceinline__ bool bit(unsigned long long bits, int r) { return ((r & 32 ? (unsigned)(bits >> 32) : (unsigned)bits) >> (r & 31)) & 1; }
// Which of the rows 32 sub + rowmap(x, h) of a tile take part: bit (x & 3) + 8 (x >> 2); `last` is the last one that this lane may see
__device__ __forceinline__ unsigned part_of(unsigned long long bits, int sub, int last, int h) {
    const unsigned word = sub ? (unsigned)(bits >> 32) : (unsigned)bits;
    const int n = last + 1 - 32 * sub;
    return (n <= 0 ? 0u : word & (~0u >> (32 - min(n, 32)))) >> (4 * h);
}
__device__ __forceinline__ unsigned all_or_none(unsigned part, int x) { return (unsigned)__builtin_amdgcn_sbfe((int)part, (x & 3) + 8 * (x >> 2), 1); }
// v where the row takes part, else `other`
__device__ __forceinline__ float where_part(unsigned part, int x, float v, float other) {
    const unsigned m = all_or_none(part, x);
    return __uint_as_float((__float_as_uint(v) & m) | (__float_as_uint(other) & ~m));
}

// ROWS x DP tiles of one tensor, global -> LDS by NT threads (a workgroup, or each wave its own).  The tile's base is the wave's, a lane adds one
// 32-bit offset (64 rows stay within 2^31 bytes: checked at the entry), so a whole tile costs no address arithmetic.  Rows whose bit is 0
// become zero; columns >= D are never written: zero_images() clears them once.
template <class T, int DP, int ROWS = KB, int NT = 256>
struct Stage {
    static constexpr int CH = Image<T, DP>::CH, N = ROWS * CH / NT, STEP = NT / CH;
    static constexpr bool EVEN = NT % CH == 0 && STEP % 16 == 0;      // round i is round 0, STEP rows further, with the same swizzle
    static_assert(ROWS * CH % NT == 0, "whole rounds");
    unsigned off[EVEN ? 1 : N];
    long long st;
    int width;                                                       // bytes of a row
    __device__ static __forceinline__ int row(int i) { return (threadIdx.x % NT + NT * i) / CH; }
    __device__ static __forceinline__ int col(int i) { return (((threadIdx.x % NT + NT * i) % CH) ^ Image<T, DP>::swz(row(i))) * 16; }
    __device__ __forceinline__ Stage(long long stride, int D) : st(stride), width(D * (int)sizeof(T)) {
#pragma unroll
        for (int i = 0; i < (EVEN ? 1 : N); ++i) off[i] = (unsigned)(row(i) * st + col(i));
    }
    __device__ __forceinline__ void issue(char* img, const char* base, unsigned long long bits) const {
        const unsigned at = lds_offset(img) + __builtin_amdgcn_readfirstlane((threadIdx.x % NT >> 6) * 1024);
        const bool all = ROWS == 64 ? bits == ~0ull : (unsigned)bits == ~0u;
        if (all && width == DP * (int)sizeof(T)) {
#pragma unroll
            for (int i = 0; i < N; ++i) copy16(EVEN ? base + i * STEP * st : base, off[EVEN ? 0 : i], at + i * NT * 16);
            return;
        }
        if (all) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (col(i) < width) copy16(EVEN ? base + i * STEP * st : base, off[EVEN ? 0 : i], at + i * NT * 16);
            return;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const char* src = base + (EVEN ? i * STEP * st : 0) + off[EVEN ? 0 : i];
            if (!bit(bits, row(i))) src = reinterpret_cast<const char*>(FILL);
            if (col(i) < width) copy16(src, at + i * NT * 16);
        }
    }
    __device__ __forceinline__ void issue_rows(char* img, const char* base, const int* rows, unsigned long long bits) const {      // (rows: in LDS)
        const unsigned at = lds_offset(img) + __builtin_amdgcn_readfirstlane((threadIdx.x % NT >> 6) * 1024);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const char* src = bit(bits, row(i)) ? base + rows[row(i)] * st + col(i) : reinterpret_cast<const char*>(FILL);
            if (col(i) < width) copy16(src, at + i * NT * 16);
        }
    }
};
__device__ __forceinline__ void zero_images(char* smem, int bytes) {  // (followed by the barrier before the first read)
    for (int i = threadIdx.x * 16; i < bytes; i += 256 * 16) *reinterpret_cast<uint4*>(smem + i) = uint4{0, 0, 0, 0};
    __syncthreads();
}
// Tiles of two tensors, one ahead: issue() starts the next one, commit() waits for it and for everyone's reads of the one before.  Copied past the
// registers into two buffers in turn (one barrier), or, split into bf16 parts, through the registers into one (two).
template <class T, int DP, int ROWS, bool S = SPLIT<T>> struct Tiles {
    static constexpr int IMG = ROWS * Image<T, DP>::PITCH, PLANE = 0, BYTES = 4 * IMG;
    char* smem;
    Stage<T, DP, ROWS> a, b;
    int next = 0, ready = 0;
    __device__ __forceinline__ Tiles(char* s, long long sta, long long stb, int D) : smem(s), a(sta, D), b(stb, D) {
        if (D < DP) zero_images(smem, BYTES);
    }
    __device__ __forceinline__ void issue(const char* pa, const char* pb, unsigned long long bits) {
        a.issue(smem + next * 2 * IMG, pa, bits);
        b.issue(smem + next * 2 * IMG + IMG, pb, bits);
    }
    __device__ __forceinline__ void issue_rows(const char* pa, const char* pb, const int* rows, unsigned long long bits) {
        a.issue_rows(smem + next * 2 * IMG, pa, rows, bits);
        b.issue_rows(smem + next * 2 * IMG + IMG, pb, rows, bits);
    }
    __device__ __forceinline__ void commit() {
        copies_done();
        __syncthreads();
        ready = next;
        next ^= 1;
    }
    __device__ __forceinline__ const char* img_a() const { return smem + ready * 2 * IMG; }
    __device__ __forceinline__ const char* img_b() const { return img_a() + IMG; }
};
template <class T, int DP, int ROWS> struct Tiles<T, DP, ROWS, true> {
    static constexpr int UNITS = DP / 8, N = ROWS * UNITS / 256, PLANE = ROWS * DP * 2, IMG = 3 * PLANE, BYTES = 2 * IMG;      // unit: 8 columns
    static_assert(ROWS * UNITS % 256 == 0, "whole rounds");
    char* smem;
    long long st[2];
    int D, next = 0, ready = 0;
    f32x4 v[2][N][2];
    __device__ __forceinline__ Tiles(char* s, long long sta, long long stb, int d) : smem(s), st{sta, stb}, D(d) {}
    __device__ __forceinline__ void issue(const char* pa, const char* pb, unsigned long long bits) {
        fetch(pa, pb, bits, [](int row, bool) { return row; });
    }
    __device__ __forceinline__ void issue_rows(const char* pa, const char* pb, const int* rows, unsigned long long bits) {
        fetch(pa, pb, bits, [&](int row, bool ok) { return ok ? rows[row] : 0; });
    }
    template <class F> __device__ __forceinline__ void fetch(const char* pa, const char* pb, unsigned long long bits, F place) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int e = threadIdx.x + 256 * i, row = e / UNITS, c = e % UNITS;
                const bool ok = bit(bits, row) && c * 8 < D;
                const f32x4* src = reinterpret_cast<const f32x4*>((t ? pb : pa) + place(row, ok) * st[t] + c * 32);
                v[t][i][0] = ok ? src[0] : f32x4{0.f, 0.f, 0.f, 0.f};
                v[t][i][1] = ok ? src[1] : f32x4{0.f, 0.f, 0.f, 0.f};
            }
    }
    __device__ __forceinline__ void commit() {
        __syncthreads();
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int e = threadIdx.x + 256 * i, row = e / UNITS, c = e % UNITS;
                const f32x4 x = v[t][i][0], y = v[t][i][1];
                const float w[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
                const Split3::Frag f = Split3::of(w);
#pragma unroll
                for (int k = 0; k < 3; ++k) *reinterpret_cast<bf16x8*>(smem + t * IMG + k * PLANE + Image<__bf16, DP>::off(row, c)) = f.p[k];
            }
        copies_done();
        __syncthreads();
        ready = next;
        next ^= 1;
    }
    __device__ __forceinline__ const char* img_a() const { return smem; }
    __device__ __forceinline__ const char* img_b() const { return smem + IMG; }
};
__device__ __forceinline__ unsigned long long first_bits(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }

// operand fragments of one row (this lane's column of the product), zero where !ok
template <class M, class T, int DP>
__device__ __forceinline__ void load_row(typename M::Frag (&f)[DP / M::KS], const char* row, int h, int D, bool ok) {
#pragma unroll
    for (int s = 0; s < DP / M::KS; ++s) {
        const int c = 2 * s + h;                                     // KS / 2 elements
        if constexpr (std::is_same_v<M, Split3>) {
            f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
            if (ok && c * 8 < D) { x = reinterpret_cast<const f32x4*>(row + c * 32)[0]; y = reinterpret_cast<const f32x4*>(row + c * 32)[1]; }
            const float w[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
            f[s] = Split3::of(w);
        } else {
            uint4 v = {0, 0, 0, 0};
            if (ok && c * 16 < D * (int)sizeof(T)) v = *reinterpret_cast<const uint4*>(row + c * 16);
            f[s] = __builtin_bit_cast(typename M::Frag, v);
        }
    }
}

// acc[dt] (rows = columns 32 dt .. of the tensor, column = this lane's row) * mul -> row
template <class T, int DP, class Q = typename Mma<T>::Quad>
__device__ __forceinline__ void store_row(const f32x16 (&acc)[DP / 32], char* row, int h, int D, float mul) {
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * dt + 8 * g + 4 * h;
            if (d < D) {
                const f32x4 v = {acc[dt][4 * g] * mul, acc[dt][4 * g + 1] * mul, acc[dt][4 * g + 2] * mul, acc[dt][4 * g + 3] * mul};
                *reinterpret_cast<Q*>(row + d * (int)(sizeof(Q) / 4)) = __builtin_convertvector(v, Q);
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
__device__ __forceinline__ float other_half(float v) {               // the value of lane l ^ 32
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(threadIdx.x & 32 ? r[0] : r[1]);
}

// fp16 only: t carries a power of two per column; where it outgrows fp16 (2^15), t and the column's sum shrink by the power of two returned.
template <int N> __device__ __forceinline__ float shrink_col(f32x16& t, f32x16 (&acc)[N]) {
    float m = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) m = fmaxf(m, fabsf(t[r]));
    m = fmaxf(m, other_half(m));
    if (!__any(m > 32768.f)) return 1.f;
    const float by = m > 32768.f ? ldexpf(1.f, 14 - min(ilogbf(m), 127)) : 1.f;
    times(acc, by);
#pragma unroll
    for (int r = 0; r < 16; ++r) t[r] *= by;
    return by;
}

// 16-bit types: sums of at most this many terms (dQ: of as many keys as a tile has) take P and dS in two parts, what the first one's rounding left being the
// second.  The terms are those of a block that take part: what a key mask leaves out does not count.  A long sum averages those roundings; one of two or four terms would be off by up to 1.6 times what a computation in 32 bits, rounded once, is.
constexpr int EXACT = 32;
// Blocks that see at most this many keys are swept for D before dQ (see there)
template <class T> constexpr int FEW_KEYS = (sizeof(T) == 2 ? 4 : 1) * KB;
template <class T> __device__ __forceinline__ constexpr bool is_f16() { return __is_same(T, _Float16); }
// Workgroups of a CU that the registers have to allow.  Rows of at most 128 bytes: three (packed fp16 24 x 1900, 12 heads of 64: forward 17 % and dQ 13 %
// faster than at two; four would spill in dQ), but for dK/dV, whose two sums would spill (5 % slower at three).  fp32: two up to head size 64, one beyond,
// whose operands of three parts fill the registers.  (fp32 dQ and dK/dV of head size 64 spill some five and some forty registers, outside of the
// innermost loops: 1 x 4096, 16 heads of 64, backward 1265 us; at one workgroup, where nothing spills, 16 % slower.)
template <class T, int DP> constexpr int WAVES = DP * sizeof(T) <= 128 ? 3 : sizeof(T) == 2 || DP <= 64 ? 2 : 1;
template <class T, int DP> constexpr int DKV_WAVES = WAVES<T, DP> < 2 ? 1 : 2;
// dK/dV at head size 128: the two sums alone take 128 registers; the values' fragments wait in LDS (V_LDS) and the staged tile has 32 rows (fp32: 146 KB
// of LDS in all)
template <class T, int DP> constexpr bool V_LDS = DP == 128;
template <class T, int DP> constexpr int RB = DP == 128 ? 32 : 64;

// The keys of a tile that take part, one tile ahead: without a key mask by the sequence's end, with one by a byte a lane
struct KeyBits {
    const unsigned char* mask;
    int kl, lane;
    unsigned char next;
    __device__ __forceinline__ void fetch(int kt) { if (mask) next = kt + lane < kl ? mask[kt + lane] : 0; }
    __device__ __forceinline__ unsigned long long bits(int kt) const { return mask ? __ballot(next != 0) : first_bits(kl - kt); }
};

// How many of the rows from .. to - 1 takes_part(row) holds for, counted until there are more than `most` (by all lanes of a wave)
template <class F> __device__ __forceinline__ int count_rows(int from, int to, int lane, int most, F takes_part) {
    int n = 0;
    for (int r0 = from; r0 < to && n <= most; r0 += 128) {
        bool in[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) in[i] = r0 + 64 * i + lane < to && takes_part(r0 + 64 * i + lane);
        n += __popcll(__ballot(in[0])) + __popcll(__ballot(in[1]));
    }
    return n;
}
// How many of the first n keys a mask lets through, counted until there are more than `most`, and the first `most` of them, in order, into `list` (LDS; four
// more words follow it).  By all 256 threads of a workgroup, 16 keys each at a time.
__device__ __forceinline__ int list_keys(const unsigned char* mask, int n, int most, int* list) {
    int* const totals = list + most;
    int live = 0;
    for (int k0 = 0; k0 < n && live <= most; k0 += 256 * 16) {
        const int k = k0 + (int)threadIdx.x * 16;
        unsigned char m[16] = {};
        if (k + 16 <= n) __builtin_memcpy(m, mask + k, 16);
        else
            for (int i = 0; i < 16; ++i) m[i] = k + i < n ? mask[k + i] : 0;
        int mine = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) mine += m[i] != 0;
        int upto = mine;                                             // of this wave, up to this thread
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) {
            const int other = __shfl_up(upto, x, 64);
            if ((int)(threadIdx.x & 63) >= x) upto += other;
        }
        __syncthreads();                                             // (the totals of the round before have been read)
        if ((threadIdx.x & 63) == 63) totals[threadIdx.x >> 6] = upto;
        __syncthreads();
        int at = live + upto - mine;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            if (w < (int)(threadIdx.x >> 6)) at += totals[w];
            live += totals[w];
        }
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (m[i] != 0) {
                if (at < most) list[at] = k + i;
                ++at;
            }
    }
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(live);
}

// What a row's sum l of exponentials, relative to 2^m, makes of it: 1 / l and the log-sum-exp; 0 and -inf for a row that saw no key.  A sum of 0 over some keys
// is none of that: scores from 2^30 on are further from their maximum by its rounding than an exponent holds, and the row becomes NaN.
__device__ __forceinline__ bool sees_none(float m, float l) { return l == 0.f && m == -INFINITY; }
__device__ __forceinline__ float inverse(float m, float l) { return sees_none(m, l) ? 0.f : 1.f / l; }
__device__ __forceinline__ float lse_of(float m, float l) {
    return l != 0.f ? (m + __builtin_amdgcn_logf(l)) * LN2 : sees_none(m, l) ? -INFINITY : __builtin_nanf("");
}

// Forward.  Rows of a query block: row r = token r / group, head kvh * group + r % group, so that heads which share keys share the tile's loads.  One
// pass over the keys with a running maximum and sum; 128 rows a workgroup, 32 a wave, tiles of 64 keys and values in two LDS buffers, one barrier a tile.
// Causal bf16 2 x 4096, 16/4 heads of 128: 152 us (900 TFLOP/s); packed causal fp16 24 x 1900, 12 heads of 64: 90 us (575); fp32 32 x 1024, 8 heads of
// 32: 209 us (165).
template <class T, int DP>
__global__ __launch_bounds__(256, (WAVES<T, DP>)) void fwd_kernel(const Params p) {
    typedef Op<T> M;
    typedef Tiles<T, DP, KB> Tl;
    constexpr int NF = DP / M::KS, NP = 32 / M::KS, ND = DP / 32;
    extern __shared__ __attribute__((aligned(16))) char smem[];       // tiles of K and V
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l31 = lane & 31, h = lane >> 5;
    const Where w = where(p, true);
    const int rows = w.ql * p.group, r0 = w.tile * QB * p.group + w.sub * QB;       // (tokens < 2^31 / 128 a sequence is far beyond memory x heads)
    if (r0 >= min(rows, (w.tile + 1) * QB * p.group)) return;
    const int off = w.kl - w.ql, rw = r0 + wave * 32, r = rw + l31;   // this wave's first row, this lane's
    const bool rok = r < rows;
    int token = rok ? r : r0;
    const int head = w.kvh * p.group + p.by_group.take(token);
    const int t_first = p.by_group(rw), t_last = p.by_group(rw + 31);   // this wave's tokens
    int kend = p.causal ? min(w.kl, min((int)p.by_group(r0 + QB - 1), w.ql - 1) + 1 + off) : w.kl, kbegin = 0;
    if (p.splits > 1) {                                              // whole tiles, at least four
        const int per = max(4, (max(kend, 0) + KB * p.splits - 1) / (KB * p.splits)) * KB;
        kbegin = w.split * per;
        kend = min(kend, kbegin + per);
    }
    const char* const kbase = p.k.p + w.b * p.k.b + w.k0 * p.k.t + w.kvh * p.k.h;
    const char* const vbase = p.v.p + w.b * p.v.b + w.k0 * p.v.t + w.kvh * p.v.h;
    KeyBits kb{p.key_mask ? p.key_mask + w.b * p.mask_b + w.k0 : nullptr, w.kl, lane, 0};
    typename M::Frag qf[NF];
    load_row<M, T, DP>(qf, p.q.p + w.b * p.q.b + (w.q0 + token) * p.q.t + head * p.q.h, h, p.D, rok);
    f32x16 o[ND];
    clear(o);
    // Exponents in powers of two.  The running maximum m is only raised when a score exceeds it by 2^8, so the sums are rarely rescaled;
    // probabilities are then at most 2^8, and fp16 carries 2^7 P on top of that so that small ones keep their bits.
    const float c = p.scale * LOG2E, lift = is_f16<T>() ? 7.f : 0.f;
    float m = -INFINITY, l = 0.f;                                    // maximum (scaled), this lane's part of the sum
    unsigned long long cur = 0;
    Tl tl(smem, p.k.t, p.v.t, p.D);
    auto issue = [&](int kt) {
        cur = kb.bits(kt);
        kb.fetch(kt + KB);                                           // (before the copies: commit() waits for all of them)
        if (cur) tl.issue(kbase + kt * p.k.t, vbase + kt * p.v.t, cur);
    };
    if (kbegin < kend) { kb.fetch(kbegin); issue(kbegin); }
    for (int kt = kbegin; kt < kend; kt += KB) {
        const unsigned long long bits = cur;
        tl.commit();
        if (kt + KB < kend) issue(kt + KB);
        if (rw >= rows || bits == 0 || (p.causal && kt > t_last + off)) continue;
        const char* const img_k = tl.img_a();
        const char* const img_v = tl.img_b();
        f32x16 st[2];
        clear(st);
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) st[sub] = M::mma(M::template row<DP, Tl::PLANE>(img_k, sub * 32 + l31, f, h), qf[f], st[sub]);
        if (bits != ~0ull || (p.causal && kt + KB - 1 > t_first + off)) {
            const int last = p.causal ? token + off - kt : KB;       // last visible key of the tile
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
                const unsigned part = part_of(bits, sub, last, h);
#pragma unroll
                for (int x = 0; x < 16; ++x) st[sub][x] = where_part(part, x, st[sub][x], -INFINITY);
            }
        }
        float tm = fmaxf(st[0][0], st[1][0]);
#pragma unroll
        for (int x = 1; x < 16; ++x) tm = fmaxf(fmaxf(tm, st[0][x]), st[1][x]);
        tm = fmaxf(tm, other_half(tm)) * c;
        if (__any(tm > m + 8.f)) {
            const float mn = fmaxf(m, tm), alpha = mn == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= alpha;
            times(o, alpha);
        }
        const float sub0 = (m == -INFINITY ? 0.f : m) - lift;
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                st[sub][x] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[sub][x], c, -sub0));
                sum[sub] += st[sub][x];
            }
        l += sum[0] + sum[1];
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
            for (int f = 0; f < NP; ++f) {
                const typename M::Frag pf = M::from_acc(st[sub], f);
#pragma unroll
                for (int dt = 0; dt < ND; ++dt) o[dt] = M::mma(M::template col<DP, Tl::PLANE>(img_v, sub * 32, f, dt, lane), pf, o[dt]);
            }
    }
    l += other_half(l);
    if (!rok) return;
    const long long at = w.b * p.lse_b + head * p.lse_h + w.q0 + token;
    if (p.splits > 1) {                                              // part: sums, part_ml [split][row][2]: maximum and sum
        const long long pr = w.split * p.part_rows + w.part(p, wave * 32 + l31);
        store_row<T, DP, f32x4>(o, reinterpret_cast<char*>(p.part + pr * p.D), h, p.D, 1.f);
        if (h == 0) {
            float* ml = p.part_ml + 2 * pr;
            ml[0] = m - lift;
            ml[1] = l;
        }
        return;
    }
    store_row<T, DP>(o, p.out.p + w.b * p.out.b + (w.q0 + token) * p.out.t + head * p.out.h, h, p.D, inverse(m, l));
    if (h == 0) p.lse[at] = lse_of(m - lift, l);
}

template <class T> __device__ __forceinline__ void store8(char* row, int d, const float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; e += 4)
        *reinterpret_cast<typename Mma<T>::Quad*>(row + (d + e) * (int)sizeof(T)) = __builtin_convertvector((f32x4{v[e], v[e + 1], v[e + 2], v[e + 3]}), typename Mma<T>::Quad);
}
// Few rows (at most 32 of a sequence and key head: single tokens, short drafts): nothing to share, so each of the four waves walks over tiles
// of 32 keys of its own, copied by itself into its own LDS, without barriers; the waves' sums are joined through LDS at the end.  Bound by the
// keys' and values' bytes: 64 KB are in flight a CU (one token, 8 x 16384 keys, 32/8 heads of 128, bf16: 100 us, 5.4 TB/s; 76 with a quarter masked).
template <class T, int DP> constexpr bool FEW = Image<T, DP>::PITCH * 32 * 16 <= 128 * 1024;
template <class T, int DP>
__global__ __launch_bounds__(256) void few_kernel(const Params p) {
    typedef Mma<T> M;
    constexpr int NF = DP / M::KS, NP = 32 / M::KS, ND = DP / 32, IMG = 32 * Image<T, DP>::PITCH, OP = DP + 4;      // OP: floats of a row of sums
    extern __shared__ __attribute__((aligned(16))) char smem[];       // [wave][2][K, V]; then [wave][32][OP] sums, [wave][32][2] maximum and sum
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l31 = lane & 31, h = lane >> 5;
    const Where w = where(p, true);
    const int rows = w.ql * p.group;                                 // <= 32: block 0 has them all
    if (w.tile * QB >= w.ql) return;
    const int off = w.kl - w.ql;
    const bool rok = l31 < rows;
    int token = rok ? l31 : 0;
    const int head = w.kvh * p.group + p.by_group.take(token);
    const int kend = p.causal ? min(w.kl, w.ql + off) : w.kl;
    const int per = (max(kend, 0) + 32 * 4 * p.splits - 1) / (32 * 4 * p.splits) * 32 * 4;       // keys of a split: whole rounds of the four waves
    const int from = w.split * per + wave * 32, to = min(kend, w.split * per + per);
    char* const mine = smem + wave * 4 * IMG;
    const char* const kbase = p.k.p + w.b * p.k.b + w.k0 * p.k.t + w.kvh * p.k.h;
    const char* const vbase = p.v.p + w.b * p.v.b + w.k0 * p.v.t + w.kvh * p.v.h;
    KeyBits kb{p.key_mask ? p.key_mask + w.b * p.mask_b + w.k0 : nullptr, w.kl, lane, 0};
    typename M::Frag qf[NF];
    load_row<M, T, DP>(qf, p.q.p + w.b * p.q.b + (w.q0 + token) * p.q.t + head * p.q.h, h, p.D, rok);
    const Stage<T, DP, 32, 64> sk(p.k.t, p.D), sv(p.v.t, p.D);
    if (p.D < DP) zero_images(smem, 16 * IMG);
    f32x16 o[ND];
    clear(o);
    const float c = p.scale * LOG2E, lift = is_f16<T>() ? 7.f : 0.f;
    float m = -INFINITY, l = 0.f;
    unsigned cur = 0;
    auto issue = [&](int kt, int buf) {
        cur = (unsigned)kb.bits(kt);
        kb.fetch(kt + 128);                                          // (before the copies: they are all waited for together)
        if (cur) {
            sk.issue(mine + buf * 2 * IMG, kbase + kt * p.k.t, cur);
            sv.issue(mine + buf * 2 * IMG + IMG, vbase + kt * p.v.t, cur);
        }
    };
    if (from < to) { kb.fetch(from); issue(from, 0); }
    int buf = 0;
    for (int kt = from; kt < to; kt += 128, buf ^= 1) {
        const unsigned bits = cur;
        copies_done();                                               // (this wave's own copies; its reads of the other buffer are in registers)
        if (kt + 128 < to) issue(kt + 128, buf ^ 1);
        if (bits == 0) continue;
        const char* const img_k = mine + buf * 2 * IMG;
        const char* const img_v = img_k + IMG;
        f32x16 st[1];
        clear(st);
#pragma unroll
        for (int f = 0; f < NF; ++f) st[0] = M::mma(M::template row<DP>(img_k, l31, f, h), qf[f], st[0]);
        if (bits != ~0u || (p.causal && kt + 31 > off)) {
            const unsigned part = part_of(bits, 0, p.causal ? token + off - kt : 32, h);
#pragma unroll
            for (int x = 0; x < 16; ++x) st[0][x] = where_part(part, x, st[0][x], -INFINITY);
        }
        float tm = st[0][0];
#pragma unroll
        for (int x = 1; x < 16; ++x) tm = fmaxf(tm, st[0][x]);
        tm = fmaxf(tm, other_half(tm)) * c;
        if (__any(tm > m + 8.f)) {
            const float mn = fmaxf(m, tm), alpha = mn == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= alpha;
            times(o, alpha);
        }
        const float sub0 = (m == -INFINITY ? 0.f : m) - lift;
#pragma unroll
        for (int x = 0; x < 16; ++x) {
            st[0][x] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[0][x], c, -sub0));
            l += st[0][x];
        }
#pragma unroll
        for (int f = 0; f < NP; ++f) {
            const typename M::Frag pf = M::from_acc(st[0], f);
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) o[dt] = M::mma(M::template col<DP>(img_v, 0, f, dt, lane), pf, o[dt]);
        }
    }
    l += other_half(l);
    __syncthreads();                                                 // (the tiles' LDS becomes the sums')
    float* const s_o = reinterpret_cast<float*>(smem);
    float2* const s_ml = reinterpret_cast<float2*>(smem + 4 * 32 * OP * sizeof(float));
    store_row<T, DP, f32x4>(o, reinterpret_cast<char*>(s_o + (wave * 32 + l31) * OP), h, p.D, 1.f);
    if (h == 0) s_ml[wave * 32 + l31] = float2{m, l};
    __syncthreads();
    const int r = tid >> 3;                                          // 8 threads a row, 16 columns each
    if (r >= rows) return;
    int rt = r;
    const int rh = w.kvh * p.group + p.by_group.take(rt);
    const long long at = w.b * p.lse_b + rh * p.lse_h + w.q0 + rt, pr = w.split * p.part_rows + w.part(p, r);
    float M0 = -INFINITY, L = 0.f, a[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) M0 = fmaxf(M0, s_ml[x * 32 + r].x);
#pragma unroll
    for (int x = 0; x < 4; ++x) {                                    // (a NaN sum counts whatever its maximum)
        const float2 ml = s_ml[x * 32 + r];
        a[x] = ml.y == 0.f ? 0.f : ml.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml.x - M0);
        L = __builtin_fmaf(ml.y, a[x], L);
    }
    const float inv = p.splits > 1 ? 1.f : inverse(M0, L);
    for (int d = (tid & 7) * 8; d < p.D; d += 64) {
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            if (a[x] == 0.f) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf(s_o[(x * 32 + r) * OP + d + e], a[x], v[e]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= inv;
        if (p.splits > 1) store8<float>(reinterpret_cast<char*>(p.part + pr * p.D), d, v);
        else store8<T>(p.out.p + w.b * p.out.b + (w.q0 + rt) * p.out.t + rh * p.out.h, d, v);
    }
    if ((tid & 7) == 0) {
        if (p.splits > 1) *reinterpret_cast<float2*>(p.part_ml + 2 * pr) = float2{M0 - lift, L};
        else p.lse[at] = lse_of(M0 - lift, L);
    }
}

// Joining the splits: 16 lanes of 8 columns a row.  Many splits: a wave a row, its four groups of lanes take a quarter of the splits each (SL = 4);
// up to 8: four rows a wave (SL = 1; the partial sums of 9990 rows in 5 splits take 5.8 us, a quarter less than with a wave a row).  A lane's loads are in flight together.
constexpr int join_slices(int splits) { return splits > 8 ? 4 : 1; }
template <int SL> struct Join {
    static constexpr int ROWS = 16 / SL;                             // of a workgroup
    int row, slice, d;
    __device__ __forceinline__ Join() : row(threadIdx.x / (16 * SL)), slice(threadIdx.x / 16 % SL), d(threadIdx.x % 16 * 8) {}
    __device__ __forceinline__ bool first() const { return slice == 0; }
    template <class F> __device__ __forceinline__ float over_slices(float v, F f) const {
        if (SL == 4) { v = f(v, __shfl_xor(v, 16, 64)); v = f(v, __shfl_xor(v, 32, 64)); }
        return v;
    }
    __device__ __forceinline__ float sum(float v) const { return over_slices(v, [](float x, float y) { return x + y; }); }
};
template <int SL, class F> __device__ __forceinline__ void join_rows(const Params& p, F f) {
    const Where w = where(p, true);                                  // (split: which ROWS rows of the block)
    const Join<SL> j;
    const int rows = w.ql * p.group, in = w.split * Join<SL>::ROWS + j.row, r = w.tile * QB * p.group + w.sub * QB + in;
    if (r >= min(rows, (w.tile + 1) * QB * p.group)) return;
    int token = r;
    const int head = w.kvh * p.group + p.by_group.take(token);
    f(w, j, token, head, w.b * p.lse_b + head * p.lse_h + w.q0 + token, w.part(p, in));
}
__device__ __forceinline__ void load8(const float* row, int d, int D, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
        const f32x4 x = d < D ? *reinterpret_cast<const f32x4*>(row + d + e) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[e + i] = x[i];
    }
}
// Sum over the splits' rows (`stride` apart), in a fixed order
template <int SL> __device__ __forceinline__ void sum_splits(const Join<SL>& j, const float* part, long long stride, int n, int D, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
#pragma unroll 4
    for (int i = j.slice; i < n; i += SL) {
        float x[8];
        load8(part + i * stride, j.d, D, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += x[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = j.sum(v[e]);
}

template <class T, int SL>
__global__ __launch_bounds__(256) void fwd_join_kernel(const Params p) {
    join_rows<SL>(p, [&](const Where& w, const Join<SL>& j, int token, int head, long long at, long long pr) {
        // the largest maximum (splits that saw nothing have -inf and sum 0; a NaN sum counts whatever its maximum: it has to come out)
        float m = -INFINITY;
#pragma unroll 4
        for (int i = j.slice; i < p.splits; i += SL) m = fmaxf(m, p.part_ml[2 * (i * p.part_rows + pr)]);
        m = j.over_slices(m, [](float x, float y) { return fmaxf(x, y); });
        float l = 0.f, v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int i = j.slice; i < p.splits; i += SL) {
            const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + 2 * (i * p.part_rows + pr));
            float x[8];
            load8(p.part + (i * p.part_rows + pr) * p.D, j.d, p.D, x);
            const float a = ml.y == 0.f ? 0.f : ml.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml.x - m);
            l = __builtin_fmaf(ml.y, a, l);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf(x[e], a, v[e]);
        }
        l = j.sum(l);
        const float inv = inverse(m, l);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = j.sum(v[e]) * inv;
        if (!j.first()) return;
        if (j.d < p.D) store8<T>(p.out.p + w.b * p.out.b + (w.q0 + token) * p.out.t + head * p.out.h, j.d, v);
        if (j.d == 0) p.lse[at] = lse_of(m, l);
    });
}

// dQ, and for the dK/dV kernel lse2 and -D.  D = sum_d dO O with the 16-bit O misses what O's rounding lost; since the probabilities of a
// row add up to 1, sum_j P (dP - D) is exactly that error, so the sweep adds it up and hands the corrected D on.  Where a block sees at most
// 256 keys -- dP and D are of one size then, and a row of one or two keys has nothing but their difference -- it is swept once for D alone
// before it is swept for dQ.  fp32 does so up to 64 keys, for the rows of few keys alone.  Seen keys are what counts, not the axis they lie on: a
// key mask's are counted first, and the few that it leaves are gathered.  Tiles, split and bound as in the forward; three products:
// 225, 146 and 278 us at its sizes (915, 535 and 185 TFLOP/s).
template <class T, int DP>
__global__ __launch_bounds__(256, (WAVES<T, DP>)) void dq_kernel(const Params p) {
    typedef Op<T> M;
    typedef Tiles<T, DP, KB> Tl;
    constexpr int NF = DP / M::KS, NP = 32 / M::KS, ND = DP / 32;
    constexpr bool FIX = sizeof(T) == 2;
    extern __shared__ __attribute__((aligned(16))) char smem[];       // tiles of K and V, then FEW_KEYS places of keys and 4 words
    int* const s_live = reinterpret_cast<int*>(smem + Tl::BYTES);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l31 = lane & 31, h = lane >> 5;
    const Where w = where(p, true);
    const int rows = w.ql * p.group, r0 = w.tile * QB * p.group + w.sub * QB;
    if (r0 >= min(rows, (w.tile + 1) * QB * p.group)) return;
    const int off = w.kl - w.ql, rw = r0 + wave * 32, r = rw + l31;
    const bool rok = r < rows;
    int token = rok ? r : r0;
    int head = w.kvh * p.group + p.by_group.take(token);
    const int t_first = p.by_group(rw), t_last = p.by_group(rw + 31);
    int kend = p.causal ? min(w.kl, min((int)p.by_group(r0 + QB - 1), w.ql - 1) + 1 + off) : w.kl, kbegin = 0;
    int kall = kend;
    const unsigned char* const mask = p.key_mask ? p.key_mask + w.b * p.mask_b + w.k0 : nullptr;
    const char* const kbase = p.k.p + w.b * p.k.b + w.k0 * p.k.t + w.kvh * p.k.h;
    const char* const vbase = p.v.p + w.b * p.v.b + w.k0 * p.v.t + w.kvh * p.v.h;
    long long at = w.b * p.lse_b + head * p.lse_h + w.q0 + token;
    const float lse = rok ? p.lse[at] : -INFINITY;
    const bool sees = lse != -INFINITY;                              // (a row that sees nothing takes no part, whatever it holds)
    const float lse2 = sees ? lse * LOG2E : INFINITY;
    typename M::Frag qf[NF], gf[NF];
    load_row<M, T, DP>(qf, p.q.p + w.b * p.q.b + (w.q0 + token) * p.q.t + head * p.q.h, h, p.D, rok);
    load_row<M, T, DP>(gf, p.dout.p + w.b * p.dout.b + (w.q0 + token) * p.dout.t + head * p.dout.h, h, p.D, rok);
    // Keys that the block sees (more than FEW_KEYS: at least that many); the rows are on their way meanwhile.  The few that a mask leaves are gathered: from
    // here on they are a sequence of their own, one split's.
    const int live = mask ? list_keys(mask, kall, FEW_KEYS<T>, s_live) : kall;
    const bool few = live <= FEW_KEYS<T>, gather = mask && few;
    int last = token + off, wave_first = t_first + off, wave_last = t_last + off;          // last key that this row, the wave's first and last row may see
    if (gather) {
        kall = live;
        last = kall - 1;
        if (p.causal) {                                              // (how many of the list lie at most at token + off)
            int n = 0;
            for (int step = FEW_KEYS<T>; step; step >>= 1) n += n + step <= kall && s_live[n + step - 1] <= token + off ? step : 0;
            last = n - 1;
        }
        wave_first = -1;
        wave_last = kall;
    }
    if (few) {
        kend = w.split == 0 ? kall : 0;
    } else if (p.splits > 1) {                                       // as in the forward
        const int per = max(4, (max(kend, 0) + KB * p.splits - 1) / (KB * p.splits)) * KB;
        kbegin = w.split * per;
        kend = min(kend, kbegin + per);
    }
    const bool kept = kall <= KB;                                    // one tile stays where it is
    KeyBits kb{gather ? nullptr : mask, gather ? live : w.kl, lane, 0};
    float nd = 0.f, rho = 0.f;                                       // -D, what D still misses (times sc)
    {
        typename M::Frag of[NF];
        load_row<M, T, DP>(of, p.out.p + w.b * p.out.b + (w.q0 + token) * p.out.t + head * p.out.h, h, p.D, rok);
        if (!sees) {
#pragma unroll
            for (int f = 0; f < NF; ++f) qf[f] = gf[f] = of[f] = typename M::Frag{};
        }
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
            for (int e = 0; e < M::KS / 2; ++e) nd = __builtin_fmaf(-M::value(of[f], e), M::value(gf[f], e), nd);
        nd += other_half(nd);
    }
    f32x16 acc[ND];
    clear(acc);
    const float c = p.scale * LOG2E;
    float sc = is_f16<T>() ? 0x1p60f : 1.f, shift = lse2 - (is_f16<T>() ? 60.f : 0.f);      // (fp16: the exponent brings the column's power of two along)
    unsigned long long cur = 0;
    Tl tl(smem, p.k.t, p.v.t, p.D);
    auto issue = [&](int kt) {
        cur = kb.bits(kt);
        kb.fetch(kt + KB);                                           // (before the copies: commit() waits for all of them)
        if (FIX && gather) tl.issue_rows(kbase, vbase, s_live + kt, cur);
        else if (cur) tl.issue(kbase + kt * p.k.t, vbase + kt * p.v.t, cur);
    };
    // P (dP - D) of the tile's keys 32 sub .. (times sc)
    auto terms = [&](f32x16& st, unsigned long long bits, int kt, int sub) {
        f32x16 dp;
#pragma unroll
        for (int x = 0; x < 16; ++x) { st[x] = 0.f; dp[x] = nd; }
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            st = M::mma(M::template row<DP, Tl::PLANE>(tl.img_a(), sub * 32 + l31, f, h), qf[f], st);
            dp = M::mma(M::template row<DP, Tl::PLANE>(tl.img_b(), sub * 32 + l31, f, h), gf[f], dp);
        }
#pragma unroll
        for (int x = 0; x < 16; ++x) st[x] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[x], c, -shift)) * dp[x];
        if (bits != ~0ull || (p.causal && kt + KB - 1 > wave_first)) {
            const unsigned part = part_of(bits, sub, p.causal ? last - kt : KB, h);
#pragma unroll
            for (int x = 0; x < 16; ++x) st[x] = where_part(part, x, st[x], 0.f);
        }
    };
    auto add = [&](const f32x16& st) {
        float a = 0.f;
#pragma unroll
        for (int x = 0; x < 16; ++x) a += st[x];
        rho += a;
    };
    auto none = [&](unsigned long long bits, int kt) { return rw >= rows || bits == 0 || (p.causal && kt > wave_last); };
    auto shrink = [&](f32x16& st) {
        if (!is_f16<T>()) return;
        const float by = shrink_col(st, acc);
        if (by != 1.f) { sc *= by; rho *= by; shift = lse2 - __builtin_amdgcn_logf(sc); }
    };
    if (!FIX && gather) {                                            // (one tile at most)
        if (kbegin < kend) tl.issue_rows(kbase, vbase, s_live, cur = kb.bits(0));
    } else if (kbegin < kend) {
        kb.fetch(kbegin);
        issue(kbegin);
    }
    if (few && kbegin < kend) {                                      // the sweep for D alone
        for (int kt = kbegin; kt < kend; kt += KB) {
            const unsigned long long bits = cur;
            tl.commit();
            if (!kept) {
                if (kt + KB >= kend) kb.fetch(kbegin);
                issue(kt + KB < kend ? kt + KB : kbegin);
            }
            if (none(bits, kt)) continue;
#pragma unroll 1
            for (int sub = 0; sub < 2; ++sub) {
                f32x16 st;
                terms(st, bits, kt, sub);
                add(st);
            }
        }
        nd -= (rho + other_half(rho)) / sc;
        rho = 0.f;
    }
    const bool parts = FIX && live <= KB;                            // (dS in two parts: see EXACT)
    for (int kt = kbegin; kt < kend; kt += KB) {
        const unsigned long long bits = cur;
        if (!kept) {
            tl.commit();
            if (kt + KB < kend) issue(kt + KB);
        }
        if (none(bits, kt)) continue;
#pragma unroll 1
        for (int sub = 0; sub < 2; ++sub) {
            f32x16 st;
            terms(st, bits, kt, sub);
            if (FIX) add(st);
            shrink(st);
#pragma unroll
            for (int f = 0; f < NP; ++f) {
                const typename M::Frag df = M::from_acc(st, f);
#pragma unroll
                for (int dt = 0; dt < ND; ++dt) acc[dt] = M::mma(M::template col<DP, Tl::PLANE>(tl.img_a(), sub * 32, f, dt, lane), df, acc[dt]);
                if constexpr (FIX)
                    if (parts) {
                        const typename M::Frag dr = M::rest(st, f, df);
#pragma unroll
                        for (int dt = 0; dt < ND; ++dt) acc[dt] = M::mma(M::template col<DP, Tl::PLANE>(tl.img_a(), sub * 32, f, dt, lane), dr, acc[dt]);
                    }
            }
        }
    }
    rho = (rho + other_half(rho)) / sc;
    if (!rok) return;
    // fp32, short of registers, works the row's place out anew, from the thread's number: kept over the loops it makes them spill (32 x 1024, 8 heads of 32:
    // 5 % slower).  16 bits keep it: 2 x 4096, 16/4 heads of 128 is 7 % slower without.
    if constexpr (sizeof(T) == 4) {
        int again = tid;
        asm volatile("" : "+v"(again));
        token = rw + (again & 31);
        head = w.kvh * p.group + p.by_group.take(token);
        at = w.b * p.lse_b + head * p.lse_h + w.q0 + token;
    }
    if (w.kl == 1) clear(acc);                                       // (the softmax of one key is constant: P (dP - D) has only rounding to give)
    const float un = p.scale / sc;
    if (p.splits > 1) {                                              // part: sums, part_ml [split][row]: rho
        const long long pr = w.split * p.part_rows + w.part(p, wave * 32 + l31);
        store_row<T, DP, f32x4>(acc, reinterpret_cast<char*>(p.part + pr * p.D), h, p.D, un);
        if (h == 0) p.part_ml[pr] = rho;
        if (h == 0 && w.split == 0) { p.lse2[at] = lse2; p.ndelta[at] = nd; }
        return;
    }
    store_row<T, DP>(acc, p.dq.p + w.b * p.dq.b + (w.q0 + token) * p.dq.t + head * p.dq.h, h, p.D, un);
    if (h == 0) { p.lse2[at] = lse2; p.ndelta[at] = nd - rho; }
}

template <class T, int SL>
__global__ __launch_bounds__(256) void dq_join_kernel(const Params p) {
    join_rows<SL>(p, [&](const Where& w, const Join<SL>& j, int token, int head, long long at, long long pr) {
        float v[8], rho = 0.f;
#pragma unroll 4
        for (int i = j.slice; i < p.splits; i += SL) rho += p.part_ml[i * p.part_rows + pr];
        rho = j.sum(rho);
        sum_splits<SL>(j, p.part + pr * p.D, p.part_rows * p.D, p.splits, p.D, v);
        if (!j.first()) return;
        if (j.d < p.D) store8<T>(p.dq.p + w.b * p.dq.b + (w.q0 + token) * p.dq.t + head * p.dq.h, j.d, v);
        if (j.d == 0) p.ndelta[at] -= rho;
    });
}

// dK and dV.  128 keys a workgroup, 32 a wave, which stay in registers (V_LDS: or LDS) with their two sums, and a walk over tiles of query rows, head
// after head of the group, so that shared heads are summed in fixed order.  Four products; lse2 and -D of a tile's rows come along into LDS and are the
// start of the accumulator.  Bound as the forward: 315, 208 and 382 us at its sizes (875, 500 and 180 TFLOP/s), the join of the first's splits 23.
template <class T, int DP>
__global__ __launch_bounds__(256, (DKV_WAVES<T, DP>)) void dkv_kernel(const Params p) {
    constexpr int R = RB<T, DP>;
    typedef Op<T> M;
    typedef Tiles<T, DP, R> Tl;
    constexpr int NF = DP / M::KS, NP = 32 / M::KS, ND = DP / 32;
    constexpr bool VL = V_LDS<T, DP>;
    constexpr int UN = DP * (int)sizeof(T) <= 128 ? 2 : 1;           // (more would spill)
    extern __shared__ __attribute__((aligned(16))) char smem[];       // tiles of Q and dO, [2][lse2, -D][64], then the waves' V fragments
    float* const s_row = reinterpret_cast<float*>(smem + Tl::BYTES);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l31 = lane & 31, h = lane >> 5;
    const Where w = where(p, false);
    if (w.tile * QB >= w.kl) return;
    const int off = w.kl - w.ql;
    const int kw = w.tile * QB + wave * 32, kj = kw + l31;           // this wave's first key, this lane's
    const bool in = kj < w.kl;
    const long long row = w.k0 + (in ? kj : 0);
    const bool live = in && (!p.key_mask || p.key_mask[w.b * p.mask_b + row]);
    typename M::Frag kf[NF], vf[NF];
    load_row<M, T, DP>(kf, p.k.p + w.b * p.k.b + row * p.k.t + w.kvh * p.k.h, h, p.D, live);
    load_row<M, T, DP>(vf, p.v.p + w.b * p.v.b + row * p.v.t + w.kvh * p.v.h, h, p.D, live);
    typename M::Frag* const s_v = reinterpret_cast<typename M::Frag*>(smem + Tl::BYTES + 1024) + wave * NF * 64 + lane;     // (each lane its own)
    if (VL) {
#pragma unroll
        for (int f = 0; f < NF; ++f) s_v[f * 64] = vf[f];
    }
    f32x16 dk[ND], dv[ND];
    clear(dk);
    clear(dv);
    const float c = p.scale * LOG2E, lift = is_f16<T>() ? 15.f : 0.f;
    float sc = is_f16<T>() ? 0x1p45f : 1.f;                          // (with the 2^15 of P: 2^60 in all)
    const int qbegin = p.causal ? max(0, w.tile * QB - off) : 0;                 // first query that sees the first key
    const int per_head = qbegin < w.ql ? (w.ql - qbegin + R - 1) / R : 0;
    int step = 0, steps = per_head * p.group;
    if (p.splits > 1) {
        const int per = (steps + p.splits - 1) / p.splits;
        step = min(steps, w.split * per);
        steps = min(steps, step + per);
    }
    const bool idle = !__any(live);                                  // (this wave's keys are all masked or behind the end)
    if (p.key_mask && !__syncthreads_or(live)) steps = step;
    // The walk: tiles of R queries, head after head.
    struct At { int head, qt; } next{w.kvh * p.group, qbegin};
    if (step < steps) { next.head += step / per_head; next.qt += step % per_head * R; }
    auto advance = [&](At a) { return a.qt + R < w.ql ? At{a.head, a.qt + R} : At{a.head + 1, qbegin}; };
    Tl tl(smem, p.q.t, p.dout.t, p.D);
    const char* const qbase = p.q.p + w.b * p.q.b + w.q0 * p.q.t;
    const char* const gbase = p.dout.p + w.b * p.dout.b + w.q0 * p.dout.t;
    const long long first_row = w.b * p.lse_b + w.q0;
    // Rows that see nothing are not read (lse = -inf; lse2 cannot tell them from rows whose lse is +inf).  Under a causal mask alone they lie before
    // qbegin; a key mask can leave any row empty, so its lse is looked at first, a tile ahead.
    float ahead = 0.f;
    auto fetch = [&](At a) {
        if (p.key_mask) ahead = a.qt + lane < w.ql ? p.lse[first_row + a.head * p.lse_h + a.qt + lane] : -INFINITY;
    };
    auto issue = [&](At a, bool more) {
        const long long at = first_row + a.head * p.lse_h + a.qt + lane;
        const unsigned long long bits = p.key_mask ? __ballot(ahead != -INFINITY) : first_bits(w.ql - a.qt);
        if (more) fetch(advance(a));                                 // (before the copies: commit() waits for all of them)
        tl.issue(qbase + a.qt * p.q.t + a.head * p.q.h, gbase + a.qt * p.dout.t + a.head * p.dout.h, bits);
        const bool there = bit(bits, lane);                          // (R = 32: the upper half is never read)
        if (wave == 0) copy4(reinterpret_cast<const char*>(there ? p.lse2 + at : FILL + 4), lds_offset(s_row + tl.next * 128));
        if (wave == 1) copy4(reinterpret_cast<const char*>(there ? p.ndelta + at : FILL), lds_offset(s_row + tl.next * 128 + 64));
    };
    At now = next;
    if (step < steps) {
        fetch(now);
        issue(now, step + 1 < steps);
        next = advance(now);
    }
    // Queries of a head that take part (more than EXACT: at least that many; asked for while the first tile is on its way)
    const int seeing = p.key_mask && sizeof(T) == 2 && step < steps
                           ? count_rows(qbegin, w.ql, lane, EXACT, [&](int i) { return p.lse[first_row + w.kvh * p.group * p.lse_h + i] != -INFINITY; })
                           : w.ql - qbegin;
    for (; step < steps; ++step) {
        const int qt = now.qt;
        tl.commit();
        if (step + 1 < steps) {
            issue(next, step + 2 < steps);
            now = next;
            next = advance(next);
        }
        if (idle || (p.causal && qt + R - 1 < kw - off)) continue;
        const char* const img_q = tl.img_a();
        const char* const img_g = tl.img_b();
        const bool partial = p.causal && kw + 31 - off > qt;
#pragma unroll UN
        for (int sub = 0; sub < R / 32; ++sub) {
            const float* const sl = s_row + tl.ready * 128 + sub * 32 + 4 * h;
            f32x16 st, dp;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 de = *reinterpret_cast<const f32x4*>(sl + 64 + 8 * g);
#pragma unroll
                for (int e = 0; e < 4; ++e) { st[4 * g + e] = 0.f; dp[4 * g + e] = de[e]; }
            }
#pragma unroll
            for (int f = 0; f < NF; ++f) {
                st = M::mma(M::template row<DP, Tl::PLANE>(img_q, sub * 32 + l31, f, h), kf[f], st);
                dp = M::mma(M::template row<DP, Tl::PLANE>(img_g, sub * 32 + l31, f, h), VL ? s_v[f * 64] : vf[f], dp);
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 le = *reinterpret_cast<const f32x4*>(sl + 8 * g);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int x = 4 * g + e;
                    float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(st[x], c, lift - le[e]));
                    if (partial && kj - off > qt + sub * 32 + rowmap(x, h)) pr = 0.f;
                    st[x] = pr;
                    dp[x] *= pr;
                }
            }
            if (is_f16<T>()) {
#pragma unroll
                for (int x = 0; x < 16; ++x) dp[x] *= sc;
                sc *= shrink_col(dp, dk);
            }
#pragma unroll
            for (int f = 0; f < NP; ++f) {
                const typename M::Frag pf = M::from_acc(st, f), df = M::from_acc(dp, f);
#pragma unroll
                for (int dt = 0; dt < ND; ++dt) {
                    dv[dt] = M::mma(M::template col<DP, Tl::PLANE>(img_g, sub * 32, f, dt, lane), pf, dv[dt]);
                    dk[dt] = M::mma(M::template col<DP, Tl::PLANE>(img_q, sub * 32, f, dt, lane), df, dk[dt]);
                }
                if constexpr (sizeof(T) == 2)
                    if (seeing <= EXACT) {
                        const typename M::Frag pr = M::rest(st, f, pf), dr = M::rest(dp, f, df);
#pragma unroll
                        for (int dt = 0; dt < ND; ++dt) {
                            dv[dt] = M::mma(M::template col<DP, Tl::PLANE>(img_g, sub * 32, f, dt, lane), pr, dv[dt]);
                            dk[dt] = M::mma(M::template col<DP, Tl::PLANE>(img_q, sub * 32, f, dt, lane), dr, dk[dt]);
                        }
                    }
            }
        }
    }
    if (!in) return;
    if (!live || w.kl == 1) clear(dk);                               // (one key: as in the dQ kernel)
    if (!live) clear(dv);
    const float un = is_f16<T>() ? 0x1p-15f : 1.f;                   // (P and with it dS carry 2^15)
    if (p.splits > 1) {                                              // part: [split][dK, dV][row][D]
        const long long pr = w.part(p, wave * 32 + l31);
        store_row<T, DP, f32x4>(dk, reinterpret_cast<char*>(p.part + ((2 * w.split) * p.part_rows + pr) * p.D), h, p.D, p.scale * un / sc);
        store_row<T, DP, f32x4>(dv, reinterpret_cast<char*>(p.part + ((2 * w.split + 1) * p.part_rows + pr) * p.D), h, p.D, un);
        return;
    }
    store_row<T, DP>(dk, p.dk.p + w.b * p.dk.b + row * p.dk.t + w.kvh * p.dk.h, h, p.D, p.scale * un / sc);
    store_row<T, DP>(dv, p.dv.p + w.b * p.dv.b + row * p.dv.t + w.kvh * p.dv.h, h, p.D, un);
}

template <class T, int SL>
__global__ __launch_bounds__(256) void dkv_join_kernel(const Params p) {
    const Where w = where(p, false);
    const Join<SL> j;
    const int in = w.split * Join<SL>::ROWS + j.row, key = w.tile * QB + in;
    if (key >= w.kl) return;
    const long long row = w.k0 + key, pr = w.part(p, in);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float v[8];
        sum_splits<SL>(j, p.part + (which * p.part_rows + pr) * p.D, 2 * p.part_rows * p.D, p.splits, p.D, v);
        const Ten& t = which ? p.dv : p.dk;
        if (j.first() && j.d < p.D) store8<T>(t.p + w.b * t.b + row * t.t + w.kvh * t.h, j.d, v);
    }
}

// p with every block in n parts (splits, or the rows that a join's workgroup has)
inline Params in_parts(Params p, int n) {
    p.by_split = Div(n);
    const int t = std::max(1, p.tiles_per_seq), per = (int)p.by_sub.d * n;
    p.band_tiles = p.causal ? (t + 3) / 4 : t;
    p.by_pair = Div(p.band_tiles * per);
    p.by_last = Div((t - (t - 1) / p.band_tiles * p.band_tiles) * per);
    p.by_band = Div(std::max(1u, p.by_pair.d * (p.pairs / 8)));
    return p;
}
inline int grid_of(const Params& p) { return p.n_tiles * p.kv_heads * (int)(p.by_sub.d * p.by_split.d); }
constexpr int JOIN = QB / Join<4>::ROWS;                             // most workgroups that join a block
#define DPC_SEQ_JOIN(kernel, p)                                                                     \
    if ((p).splits > 1) {                                                                            \
        const bool many = join_slices((p).splits) == 4;                                              \
        const Params j = in_parts(p, QB / (many ? Join<4>::ROWS : Join<1>::ROWS));                   \
        if (many) hipLaunchKernelGGL((kernel<T, 4>), dim3(grid_of(j)), dim3(256), 0, s, j);          \
        else hipLaunchKernelGGL((kernel<T, 1>), dim3(grid_of(j)), dim3(256), 0, s, j);               \
        DPC_LAUNCH_CHECK();                                                                          \
    }

template <class T, int DP>
int run_fwd(const Params& p, hipStream_t s) {
    constexpr int lds = Tiles<T, DP, KB>::BYTES;
    if constexpr (FEW<T, DP>) {
        if (p.few) {
            constexpr int lds_few = std::max(16 * 32 * Image<T, DP>::PITCH, 4 * 32 * ((DP + 4) * 4 + 8));
            static DeviceOnce few;
            if (!few) { DPC_HIP(hipFuncSetAttribute((const void*)few_kernel<T, DP>, hipFuncAttributeMaxDynamicSharedMemorySize, lds_few)); few = true; }
            hipLaunchKernelGGL((few_kernel<T, DP>), dim3(grid_of(p)), dim3(256), lds_few, s, p);
        }
    }
    if (!p.few) {
        static DeviceOnce once;
        if (!once) { DPC_HIP(hipFuncSetAttribute((const void*)fwd_kernel<T, DP>, hipFuncAttributeMaxDynamicSharedMemorySize, lds)); once = true; }
        hipLaunchKernelGGL((fwd_kernel<T, DP>), dim3(grid_of(p)), dim3(256), lds, s, p);
    }
    DPC_LAUNCH_CHECK();
    DPC_SEQ_JOIN(fwd_join_kernel, p)
    return DPC_OK;
}

template <class T, int DP>
int run_bwd(const Params& pq, const Params& pk, hipStream_t s) {
    constexpr int lds = Tiles<T, DP, KB>::BYTES + (FEW_KEYS<T> + 4) * (int)sizeof(int), lds_k = Tiles<T, DP, RB<T, DP>>::BYTES + 1024 + (V_LDS<T, DP> ? 256 * (DP / Op<T>::KS) * (int)sizeof(typename Op<T>::Frag) : 0);
    static_assert(lds_k <= 160 * 1024, "LDS of a CU");
    static DeviceOnce once;
    if (!once) {
        DPC_HIP(hipFuncSetAttribute((const void*)dq_kernel<T, DP>, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
        DPC_HIP(hipFuncSetAttribute((const void*)dkv_kernel<T, DP>, hipFuncAttributeMaxDynamicSharedMemorySize, lds_k));
        once = true;
    }
    if (pq.n_tiles) {
        hipLaunchKernelGGL((dq_kernel<T, DP>), dim3(grid_of(pq)), dim3(256), lds, s, pq);
        DPC_LAUNCH_CHECK();
        DPC_SEQ_JOIN(dq_join_kernel, pq)
    }
    if (pk.n_tiles) {
        hipLaunchKernelGGL((dkv_kernel<T, DP>), dim3(grid_of(pk)), dim3(256), lds_k, s, pk);
        DPC_LAUNCH_CHECK();
        DPC_SEQ_JOIN(dkv_join_kernel, pk)
    }
    return DPC_OK;
}

// one element type's kernels live in one translation unit (seq_attn_{f32,f16,bf16}.hip)
template <class T> int fwd(const Params& p, hipStream_t s) {
    return p.D <= 32 ? run_fwd<T, 32>(p, s) : p.D <= 64 ? run_fwd<T, 64>(p, s) : p.D <= 96 ? run_fwd<T, 96>(p, s) : run_fwd<T, 128>(p, s);
}
template <class T> int bwd(const Params& pq, const Params& pk, hipStream_t s) {
    return pq.D <= 32 ? run_bwd<T, 32>(pq, pk, s) : pq.D <= 64 ? run_bwd<T, 64>(pq, pk, s) : pq.D <= 96 ? run_bwd<T, 96>(pq, pk, s) : run_bwd<T, 128>(pq, pk, s);
}
int fwd_f32(const Params&, hipStream_t);
int fwd_f16(const Params&, hipStream_t);
int fwd_bf16(const Params&, hipStream_t);
int bwd_f32(const Params&, const Params&, hipStream_t);
int bwd_f16(const Params&, const Params&, hipStream_t);
int bwd_bf16(const Params&, const Params&, hipStream_t);

}  // namespace seqattn
}  // namespace dpc
