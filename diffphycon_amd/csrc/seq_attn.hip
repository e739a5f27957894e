// Entry points of the attention on token sequences (include/dpc.h: dpc_seq_attn); the kernels are in seq_attn.h.
#include <algorithm>
#include <cmath>

#include "seq_attn.h"

namespace dpc {
namespace seqattn {

constexpr long long MAX_TOKEN_STRIDE = ((1ll << 31) - 4096) / 64;    // bytes: 64 rows within 2^31, for a lane's offset in a tile is 32 bits

constexpr long long MAX_KEYS = (1ll << 31) - (1 << 17);             // keys are counted in 32 bits, up to 128 times 512 splits behind the last one

static bool bad_tensor(const dpc_seq_tensor& t, int es) {
    return !t.p || ((size_t)t.p | (size_t)(t.stride_b * es) | (size_t)(t.stride_t * es) | (size_t)(t.stride_h * es)) % 16 != 0 ||
           t.stride_t < 0 || t.stride_t * es > MAX_TOKEN_STRIDE;
}

static int check(const dpc_seq_attn* a, bool backward) {
    DPC_REQUIRE(a, "seq_attn: null argument");
    DPC_REQUIRE(a->type >= DPC_SEQ_F32 && a->type <= DPC_SEQ_BF16, "seq_attn: unknown element type");
    DPC_REQUIRE(a->batch >= 0 && a->q_len >= 0 && a->k_len >= 0, "seq_attn: negative size");
    DPC_REQUIRE(a->heads >= 1 && a->kv_heads >= 1 && a->heads % a->kv_heads == 0, "seq_attn: heads must be a multiple of kv_heads");
    DPC_REQUIRE(a->head_dim >= 8 && a->head_dim <= 128 && a->head_dim % 8 == 0, "seq_attn: head_dim must be a multiple of 8 up to 128");
    DPC_REQUIRE((a->q_len + 2ll * QB) * (a->heads / a->kv_heads) < (1ll << 31) && a->k_len <= MAX_KEYS, "seq_attn: sequence too long");
    DPC_REQUIRE(a->scale > 0.f && std::isfinite(a->scale), "seq_attn: scale must be positive and finite");
    DPC_REQUIRE(!a->q_tiles == !a->k_tiles && a->n_q_tiles >= 0 && a->n_k_tiles >= 0 && (a->q_tiles || a->n_q_tiles + a->n_k_tiles == 0) &&
                    ((size_t)a->q_tiles | (size_t)a->k_tiles) % 32 == 0, "seq_attn: both block lists, on 32 bytes, or neither");
    if (a->batch == 0) return DPC_OK;
    const int es = a->type == DPC_SEQ_F32 ? 4 : 2;
    const char* msg = "seq_attn: tensors must not be null; bases and strides must be multiples of 16 bytes, token strides at most 2^25 - 64 bytes";
    if (a->q_len) DPC_REQUIRE(!bad_tensor(a->q, es) && !bad_tensor(a->out, es) && a->lse, msg);
    if (a->q_len && a->k_len) DPC_REQUIRE(!bad_tensor(a->k, es) && !bad_tensor(a->v, es), msg);
    if (backward) {
        if (a->q_len) DPC_REQUIRE(!bad_tensor(a->dout, es) && !bad_tensor(a->dq, es), msg);
        if (a->k_len) DPC_REQUIRE(!bad_tensor(a->dk, es) && !bad_tensor(a->dv, es), msg);
        if (a->k_len && a->q_len == 0) DPC_REQUIRE(!bad_tensor(a->k, es) && !bad_tensor(a->v, es), msg);
    }
    return DPC_OK;
}

static Params params(const dpc_seq_attn* a) {
    const long long es = a->type == DPC_SEQ_F32 ? 4 : 2;
    auto ten = [&](const dpc_seq_tensor& t) { return Ten{(char*)t.p, t.stride_b * es, t.stride_t * es, t.stride_h * es}; };
    Params p{};
    p.q = ten(a->q); p.k = ten(a->k); p.v = ten(a->v); p.out = ten(a->out);
    p.dout = ten(a->dout); p.dq = ten(a->dq); p.dk = ten(a->dk); p.dv = ten(a->dv);
    p.lse = a->lse; p.lse_b = a->lse_stride_b; p.lse_h = a->lse_stride_h;
    p.key_mask = a->key_mask; p.mask_b = a->mask_stride_b;
    p.heads = a->heads; p.kv_heads = a->kv_heads; p.group = a->heads / a->kv_heads; p.D = a->head_dim;
    p.q_len = a->q_len; p.k_len = a->k_len; p.causal = a->causal != 0; p.scale = a->scale;
    return p;
}

// Blocks and splits.  A CU holds two workgroups, the card 512.  Where the blocks alone do not fill 3/4 of them, the axis that a block walks
// along (keys; for dK/dV the query rows of the group) is split over as many workgroups as fit, each with at least four tiles to walk;
// the partial sums are joined in order by a second launch.  Under a causal mask over (nearly) square scores the blocks' walks differ by the
// length of the sequence and the longest one decides while all are resident: twice as many workgroups are made, and the card evens them out (dK/dV of
// causal bf16 2 x 4096, 16/4 heads of 128: 28 % less with its join of 23 us, which was 14).
// Returns false when a launch would have 2^32 threads or more.
constexpr int SLOTS = 512;
static bool plan_grid(Params& p, const dpc_seq_attn* a, bool keys, bool forward) {
    p.tiles = keys ? a->k_tiles : a->q_tiles;
    p.tiles_per_seq = cdiv(keys ? a->k_len : a->q_len, QB);
    const long long n = p.tiles ? (keys ? a->n_k_tiles : a->n_q_tiles) : (long long)a->batch * p.tiles_per_seq;
    const int subs = keys ? 1 : std::max(1, cdiv((long long)std::min(a->q_len, QB) * p.group, QB));
    const long long blocks = n * p.kv_heads * subs;
    const long long walk = keys ? (long long)p.group * cdiv(a->q_len, KB) : cdiv(a->k_len, KB);
    const int slots = p.causal && 2ll * a->q_len > a->k_len ? 2 * SLOTS : SLOTS;
    // At most 32 rows of a sequence and key head: few_kernel (its LDS allows rows of 256 bytes), as many workgroups as are resident at once -- one a CU, two with
    // rows of 128 bytes -- for each starts with empty loads in flight; a split has two tiles a wave at least.  One token, 32/8 heads of 128, bf16, against
    // 512 workgroups: 8 x 16384 keys 3 % faster, a quarter of them masked 16 %, 1 x 16384 keys 20 %; fwd_kernel takes 12 % longer for the first.
    const int row = (a->head_dim + 31) / 32 * 32 * (a->type == DPC_SEQ_F32 ? 4 : 2);
    p.few = forward && (long long)a->q_len * p.group <= 32 && row <= 256;
    if (p.few) p.splits = blocks == 0 ? 1 : (int)std::max<long long>(1, std::min<long long>((row <= 128 ? SLOTS : SLOTS / 2) / blocks, a->k_len / 256));
    else p.splits = blocks == 0 || blocks >= slots * 3 / 4 ? 1 : (int)std::max<long long>(1, std::min<long long>(slots / blocks, walk / 4));
    p.n_tiles = (int)n;
    p.pairs = a->batch * p.kv_heads;
    p.by_sub = Div(subs); p.by_kv = Div(p.kv_heads); p.by_group = Div(p.group); p.by_tile = Div(std::max(1, p.pairs));
    p = in_parts(p, p.splits);
    p.block_rows = keys ? std::min(a->k_len, QB) : (int)std::min<long long>((long long)a->q_len * p.group, QB);
    p.part_rows = blocks * p.block_rows;
    return n < (1ll << 31) && blocks * (p.splits > 1 ? std::max(p.splits, JOIN) : 1) < (1ll << 24);
}

static size_t part_bytes(const Params& p, int per_row) {
    return p.splits > 1 ? align_up((size_t)p.splits * p.part_rows * per_row * sizeof(float), 256) : 0;
}

struct Plan { Params q, k; size_t rows, bytes; bool ok; };
static Plan plan_of(const dpc_seq_attn* a, bool backward) {
    Plan w{};
    w.q = params(a);
    w.k = w.q;
    w.ok = plan_grid(w.q, a, false, !backward) && (!backward || plan_grid(w.k, a, true, false));
    if (backward) {
        w.rows = align_up((size_t)a->lse_rows * sizeof(float), 256);
        w.bytes = 2 * w.rows + std::max(part_bytes(w.q, a->head_dim + 1), part_bytes(w.k, 2 * a->head_dim));
    } else {
        w.bytes = part_bytes(w.q, a->head_dim + 2);
    }
    if (w.bytes) w.bytes += 256;
    return w;
}

}  // namespace seqattn
}  // namespace dpc

using namespace dpc;
using namespace dpc::seqattn;

extern "C" {

size_t dpc_seq_attn_workspace_bytes(const dpc_seq_attn* a, int backward) {
    if (check(a, backward != 0) != DPC_OK || a->batch == 0) return 0;
    return plan_of(a, backward != 0).bytes;
}

int dpc_seq_attn_fwd(const dpc_seq_attn* a, void* ws, size_t ws_bytes, dpc_stream_t stream) {
    const int rc = check(a, false);
    if (rc != DPC_OK) return rc;
    if (a->batch == 0) return DPC_OK;
    Plan w = plan_of(a, false);
    DPC_REQUIRE(w.ok, "seq_attn: grid too large");
    DPC_REQUIRE(w.bytes == 0 || (ws && ws_bytes >= w.bytes), "seq_attn: workspace too small");
    if (w.q.n_tiles == 0) return DPC_OK;
    w.q.part = reinterpret_cast<float*>(align_up((size_t)ws, 256));
    w.q.part_ml = w.q.part + (size_t)w.q.splits * w.q.part_rows * a->head_dim;
    hipStream_t s = (hipStream_t)stream;
    ProfScope prof(PROF_ATTN, 4.0 * a->batch * a->heads * (double)a->q_len * a->k_len * a->head_dim, 0, s);
    return a->type == DPC_SEQ_F32 ? fwd_f32(w.q, s) : a->type == DPC_SEQ_F16 ? fwd_f16(w.q, s) : fwd_bf16(w.q, s);
}

int dpc_seq_attn_bwd(const dpc_seq_attn* a, void* ws, size_t ws_bytes, dpc_stream_t stream) {
    const int rc = check(a, true);
    if (rc != DPC_OK) return rc;
    if (a->batch == 0) return DPC_OK;
    Plan w = plan_of(a, true);
    DPC_REQUIRE(w.ok, "seq_attn_bwd: grid too large");
    DPC_REQUIRE(w.bytes == 0 || (ws && ws_bytes >= w.bytes), "seq_attn_bwd: workspace too small");
    const size_t base = align_up((size_t)ws, 256);
    for (Params* p : {&w.q, &w.k}) {
        p->lse2 = reinterpret_cast<float*>(base);
        p->ndelta = reinterpret_cast<float*>(base + w.rows);
        p->part = reinterpret_cast<float*>(base + 2 * w.rows);
        p->part_ml = p->part + (size_t)p->splits * p->part_rows * a->head_dim;
    }
    hipStream_t s = (hipStream_t)stream;
    ProfScope prof(PROF_ATTN_BWD, 10.0 * a->batch * a->heads * (double)a->q_len * a->k_len * a->head_dim, 0, s);
    return a->type == DPC_SEQ_F32 ? bwd_f32(w.q, w.k, s) : a->type == DPC_SEQ_F16 ? bwd_f16(w.q, w.k, s) : bwd_bf16(w.q, w.k, s);
}

}  // extern "C"
