// Entry points of the attention on token sequences (include/dpc.h: dpc_seq_attn); the kernels are in seq_attn.h.
#include <cmath>

#include "seq_attn.h"

namespace dpc {
namespace seqattn {

static bool bad_tensor(const dpc_seq_tensor& t, int es) {
    return !t.p || ((size_t)t.p | (size_t)(t.stride_b * es) | (size_t)(t.stride_t * es) | (size_t)(t.stride_h * es)) % 16 != 0;
}

static int check(const dpc_seq_attn* a, bool backward) {
    DPC_REQUIRE(a, "seq_attn: null argument");
    DPC_REQUIRE(a->type >= DPC_SEQ_F32 && a->type <= DPC_SEQ_BF16, "seq_attn: unknown element type");
    DPC_REQUIRE(a->batch >= 0 && a->q_len >= 0 && a->k_len >= 0, "seq_attn: negative size");
    DPC_REQUIRE(a->heads >= 1 && a->kv_heads >= 1 && a->heads % a->kv_heads == 0, "seq_attn: heads must be a multiple of kv_heads");
    DPC_REQUIRE(a->head_dim >= 8 && a->head_dim <= 128 && a->head_dim % 8 == 0, "seq_attn: head_dim must be a multiple of 8 up to 128");
    DPC_REQUIRE(a->scale > 0.f && std::isfinite(a->scale), "seq_attn: scale must be positive and finite");
    DPC_REQUIRE(!a->seqs || ((a->q_tiles || !a->n_q_tiles) && (a->k_tiles || !a->n_k_tiles) && a->n_q_tiles >= 0 && a->n_k_tiles >= 0),
                "seq_attn: sequences need their block lists");
    if (a->batch == 0) return DPC_OK;
    const int es = a->type == DPC_SEQ_F32 ? 4 : 2;
    const char* msg = "seq_attn: tensors must not be null; bases and strides must be multiples of 16 bytes";
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
    p.seqs = a->seqs;
    p.heads = a->heads; p.kv_heads = a->kv_heads; p.group = a->heads / a->kv_heads; p.D = a->head_dim;
    p.q_len = a->q_len; p.k_len = a->k_len; p.causal = a->causal; p.scale = a->scale;
    return p;
}

// workgroups of a kernel that walks over blocks of QB rows; < 0: too many
static int blocks(Params& p, const dpc_seq_attn* a, bool keys) {
    p.tiles = a->seqs ? (keys ? a->k_tiles : a->q_tiles) : nullptr;
    p.tiles_per_seq = cdiv(keys ? a->k_len : a->q_len, QB);
    const long long n = (a->seqs ? (keys ? a->n_k_tiles : a->n_q_tiles) : (long long)a->batch * p.tiles_per_seq) * (keys ? a->kv_heads : a->heads);
    return n < (1ll << 31) ? (int)n : -1;
}

}  // namespace seqattn
}  // namespace dpc

using namespace dpc;
using namespace dpc::seqattn;

extern "C" {

size_t dpc_seq_attn_workspace_bytes(const dpc_seq_attn* a, int backward) {
    if (!a || !backward || a->lse_rows <= 0) return 256;
    return 2 * align_up((size_t)a->lse_rows * sizeof(float), 256) + 256;
}

int dpc_seq_attn_fwd(const dpc_seq_attn* a, void* ws, size_t ws_bytes, dpc_stream_t stream) {
    const int rc = check(a, false);
    if (rc != DPC_OK) return rc;
    (void)ws; (void)ws_bytes;
    Params p = params(a);
    const int grid = blocks(p, a, false);
    DPC_REQUIRE(grid >= 0, "seq_attn: grid too large");
    if (grid == 0) return DPC_OK;
    hipStream_t s = (hipStream_t)stream;
    ProfScope prof(PROF_ATTN, 4.0 * a->batch * a->heads * (double)a->q_len * a->k_len * a->head_dim, 0, s);
    return a->type == DPC_SEQ_F32 ? fwd_f32(p, grid, s) : a->type == DPC_SEQ_F16 ? fwd_f16(p, grid, s) : fwd_bf16(p, grid, s);
}

int dpc_seq_attn_bwd(const dpc_seq_attn* a, void* ws, size_t ws_bytes, dpc_stream_t stream) {
    const int rc = check(a, true);
    if (rc != DPC_OK) return rc;
    if (a->batch == 0) return DPC_OK;
    DPC_REQUIRE(a->q_len == 0 || (ws && ws_bytes >= dpc_seq_attn_workspace_bytes(a, 1)), "seq_attn_bwd: workspace too small");
    Params p = params(a);
    p.lse2 = reinterpret_cast<float*>(align_up((size_t)ws, 256));
    p.delta = reinterpret_cast<float*>(align_up((size_t)ws, 256) + align_up((size_t)a->lse_rows * sizeof(float), 256));
    Params pk = p;
    const int gq = blocks(p, a, false), gk = blocks(pk, a, true);
    DPC_REQUIRE(gq >= 0 && gk >= 0, "seq_attn_bwd: grid too large");
    hipStream_t s = (hipStream_t)stream;
    ProfScope prof(PROF_ATTN_BWD, 10.0 * a->batch * a->heads * (double)a->q_len * a->k_len * a->head_dim, 0, s);
    return a->type == DPC_SEQ_F32 ? bwd_f32(p, gq, pk, gk, s) : a->type == DPC_SEQ_F16 ? bwd_f16(p, gq, pk, gk, s) : bwd_bf16(p, gq, pk, gk, s);
}

}  // extern "C"
