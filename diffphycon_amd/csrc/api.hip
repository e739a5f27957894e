// extern "C" surface of libdpc (see include/dpc.h): error plumbing and the operator-level entry points.
#include <atomic>
#include <map>
#include <memory>
#include <mutex>
#include <tuple>
#include <vector>

#include "common.h"

namespace dpc {
static thread_local std::string g_err;
void set_error(const std::string& msg) { g_err = msg; }
int fail(int code, const std::string& msg) {
    g_err = msg;
    return code;
}

// ---------------------------------------------------------------- arithmetic modes
static int parse_mode(const char* e, int dflt) {
    if (!e || !e[0]) return dflt;
    if ((e[0] == 'f' || e[0] == 'F') && e[1] == '3') return 0;                  // "f32"
    if (e[0] == 'x' || e[0] == 'X' || e[0] == 'b' || e[0] == 'B') return 1;      // "x6" / "bf16x6"
    if ((e[0] == 'f' || e[0] == 'F' || e[0] == 'h') && e[1] == '1') return 2;   // "f16x3"
    return -1;
}
static Modes& global_modes_ref() {
    static Modes m = [] {
        Modes v;
        auto rd = [](const char* name) { const int r = parse_mode(getenv(name), 2); return r < 0 ? 2 : r; };
        v.conv = rd("DPC_CONV_MODE"); v.igemm = rd("DPC_IGEMM_MODE"); v.attn = rd("DPC_ATTN_MODE"); v.stem = rd("DPC_STEM_MODE");
        return v;
    }();
    return m;
}
static thread_local const Modes* g_scope = nullptr;
Modes modes_global() { return global_modes_ref(); }
const Modes& modes_current() { return g_scope ? *g_scope : global_modes_ref(); }
ModeScope::ModeScope(const Modes& m) : prev_(g_scope), cur_(m) { g_scope = &cur_; }
ModeScope::~ModeScope() { g_scope = prev_; }
const char* mode_name(int mode) { return mode == 0 ? "f32" : (mode == 1 ? "x6" : "f16x3"); }
std::string modes_string(const Modes& m) {
    return std::string("conv=") + mode_name(m.conv) + ",igemm=" + mode_name(m.igemm) + ",attn=" + mode_name(m.attn) +
           ",stem=" + mode_name(m.stem);
}
static thread_local RangeCheck* g_range = nullptr;
RangeCheck* range_check_current() { return g_range; }
RangeCheckScope::RangeCheckScope(RangeCheck* rc) : prev_(g_range) { g_range = rc; }
RangeCheckScope::~RangeCheckScope() { g_range = prev_; }
static thread_local int* g_oflow = nullptr;
int* overflow_flag_current() { return g_oflow; }
OverflowScope::OverflowScope(int* flag) : prev_(g_oflow) { g_oflow = flag; }
OverflowScope::~OverflowScope() { g_oflow = prev_; }
int range_check_note(const float* a0, long long rows0, int C0, const float* a1, long long rows1, int C1, const float* in_coef,
                     long long rows_per_sample, hipStream_t s) {
    RangeCheck* rc = g_range;
    if (!rc || !rc->on || !rc->flag) return DPC_OK;
    rc->names.push_back(rc->cur);
    const int id = (int)rc->names.size();
    const float limit = 65504.f / 16.f;
    if (a0 && C0 > 0)
        if (int r = launch_range_check(a0, rows0, C0, in_coef, rows_per_sample, limit, rc->flag, id, s)) return r;
    if (a1 && C1 > 0)
        if (int r = launch_range_check(a1, rows1, C1, nullptr, 0, limit, rc->flag, id, s)) return r;
    return DPC_OK;
}
int debug_switch(const char* name, int dflt) {
    static const bool on = [] { const char* e = getenv("DPC_DEBUG"); return e && e[0] == '1'; }();
    if (!on) return dflt;
    const char* e = getenv(name);
    return e ? atoi(e) : dflt;
}
// Library-internal scratch keyed by (slot, device, stream): work enqueued on ONE stream is ordered, so two launches that share a
// buffer of this table can never overlap; different streams (DPC_TWO_STREAMS, a multi-threaded C-ABI user) get different buffers.
// Grown geometrically under a mutex; a superseded allocation stays alive in `old` (a captured HIP graph may still replay kernels
// that hold its address) and is released with the process.
static thread_local void* g_scratch_base = nullptr;
static thread_local size_t g_scratch_bytes = 0;
ScratchScope::ScratchScope(void* base, size_t bytes) : prev_base_(g_scratch_base), prev_bytes_(g_scratch_bytes) {
    g_scratch_base = base;
    g_scratch_bytes = base ? bytes : 0;
}
ScratchScope::~ScratchScope() { g_scratch_base = prev_base_; g_scratch_bytes = prev_bytes_; }
int stream_scratch(int slot, hipStream_t s, size_t bytes, float** out) {
    if (g_scratch_base && bytes <= g_scratch_bytes) {        // a U-Net forward lent a region of ITS workspace (graph-capture safe)
        *out = static_cast<float*>(g_scratch_base);
        return DPC_OK;
    }
    struct Entry { void* p = nullptr; size_t cap = 0; };
    static std::mutex mu;
    static std::map<std::tuple<int, int, hipStream_t>, Entry> table;
    static std::vector<void*> old;
    int dev = 0;
    (void)hipGetDevice(&dev);
    std::lock_guard<std::mutex> lock(mu);
    Entry& e = table[std::make_tuple(slot, dev, s)];
    if (bytes > e.cap) {
        const size_t want = std::max(bytes, 2 * e.cap);
        void* fresh = nullptr;
        DPC_HIP(hipMalloc(&fresh, want));
        if (e.p) old.push_back(e.p);
        e.p = fresh;
        e.cap = want;
    }
    *out = static_cast<float*>(e.p);
    return DPC_OK;
}
// CU budget of the persistent kernels (dpc_set_cu_budget): the grids of conv3w / conv3f3c / tattn3 are "one workgroup per CU"; while a
// long-running kernel of ANOTHER stream occupies some CUs (the smoke evaluator: one 129 KB-LDS workgroup per rollout), a full-size
// grid would leave workgroups waiting for a CU and their statically assigned tiles would run as a second round.
static std::atomic<int> g_cu_budget{0};
int cu_budget(int ncu) {
    const int b = g_cu_budget.load(std::memory_order_relaxed);
    return (b > 0 && b < ncu) ? std::max(8, b / 8 * 8) : ncu;
}
int conv_mode_default() { return modes_current().conv; }
int igemm_mode_default() { return modes_current().igemm; }
}  // namespace dpc

using namespace dpc;

extern "C" {

int dpc_version(void) { return 103; }
int dpc_set_cu_budget(int cus) {
    DPC_REQUIRE(cus >= 0, "set_cu_budget: negative");
    g_cu_budget.store(cus, std::memory_order_relaxed);
    return DPC_OK;
}
const char* dpc_last_error(void) { return g_err.c_str(); }

int dpc_set_mode(const char* family, const char* mode) {
    DPC_REQUIRE(family && mode, "set_mode: null argument");
    const int m = parse_mode(mode, -1);
    DPC_REQUIRE(m >= 0, std::string("set_mode: unknown mode '") + mode + "' (f32 | x6 | f16x3)");
    Modes& g = global_modes_ref();
    const std::string f(family);
    if (f == "conv") g.conv = m;
    else if (f == "igemm") g.igemm = m;
    else if (f == "attn") g.attn = m;
    else if (f == "stem") g.stem = m;
    else if (f == "all") g.conv = g.igemm = g.attn = g.stem = m;
    else return fail(DPC_ERR_ARG, "set_mode: unknown op family '" + f + "' (conv | igemm | attn | stem | all)");
    return DPC_OK;
}

const char* dpc_get_mode(const char* family) {
    static thread_local std::string buf;
    const Modes g = modes_global();
    const std::string f(family ? family : "all");
    if (f == "conv") return mode_name(g.conv);
    if (f == "igemm") return mode_name(g.igemm);
    if (f == "attn") return mode_name(g.attn);
    if (f == "stem") return mode_name(g.stem);
    buf = modes_string(g);
    return buf.c_str();
}

const char* dpc_conv3d_algorithm(void) { return !conv3w_shape_ok(4, 8, 8, 64, 64) ? "direct" : conv3w_f43_enabled() ? "winograd_f43_frames" : "winograd_f23_frames"; }

int dpc_ddpm_update_smoke(const float* x, const float* eps_j, const float* eps_w, const float* z, const float* init,
                          const float* rescaler, float* x_next, float* x0_out, const dpc_step_coef* coef, int B,
                          int F, int C, int H, int W, dpc_stream_t stream) {
    DPC_REQUIRE(x && eps_j && eps_w && init && rescaler && x_next && coef, "ddpm_update_smoke: null argument");
    DPC_REQUIRE(B >= 0 && F >= 1 && H >= 1 && W >= 1, "ddpm_update_smoke: bad shape");
    return launch_ddpm_update_smoke(x, eps_j, eps_w, z, init, rescaler, x_next, x0_out, *coef, B, F, C, H, W,
                                    (hipStream_t)stream);
}

int dpc_burgers_prepare(float* img, float* x_w, const float* u0, const float* uT, int B, int nt, int nx, int cond_idx,
                        int set_zero, dpc_stream_t stream) {
    DPC_REQUIRE(img && B >= 0 && nt >= 2 && nx >= 4 && cond_idx >= 1 && cond_idx < nt, "burgers_prepare: bad argument");
    return launch_burgers_prepare(img, x_w, u0, uT, B, nt, nx, cond_idx, set_zero, (hipStream_t)stream);
}

int dpc_ddpm_update_burgers(const float* x, const float* eps_uw, const float* eps_w, const float* z,
                            const float* u_target, float* x_next, float* x0_out, float* eps_out,
                            const dpc_burgers_coef* coef, int B, int nt, int nx, dpc_stream_t stream) {
    DPC_REQUIRE(x && eps_uw && x_next && coef && B >= 0 && nt >= 2 && nx >= 4, "ddpm_update_burgers: bad argument");
    return launch_ddpm_update_burgers(x, eps_uw, eps_w, z, u_target, x_next, x0_out, eps_out, *coef, B, nt, nx,
                                      (hipStream_t)stream);
}

int dpc_ddpm_update_jelly(const float* x, const float* eps, const float* eps_guided, const float* z, float* pred,
                          float* x0_out, const dpc_jelly_coef* coef, int B, int F, int Cx, int n_state, int H, int W,
                          dpc_stream_t stream) {
    DPC_REQUIRE(x && eps && pred && coef && B >= 0 && F >= 1 && H >= 1 && W >= 1, "ddpm_update_jelly: bad argument");
    return launch_ddpm_update_jelly(x, eps, eps_guided, z, pred, x0_out, *coef, B, F, Cx, n_state, H, W, (hipStream_t)stream);
}

int dpc_jelly_apply_guidance(float* io, const float* g, const float* eps_w, float eta_J, float eta_w, int pad_w,
                             float sign, int B, int F, int Cd, int H, int W, dpc_stream_t stream) {
    DPC_REQUIRE(io && B >= 0 && F >= 1 && Cd >= 1 && H >= 1 && W >= 1, "jelly_apply_guidance: bad argument");
    return launch_jelly_guidance(io, g, eps_w, eta_J, eta_w, pad_w, sign, B, F, Cd, H, W, (hipStream_t)stream);
}

int dpc_philox_normal(float* out, int B, int64_t per_traj, uint64_t seed, int64_t traj0, int64_t draw,
                      dpc_stream_t stream) {
    DPC_REQUIRE(out && B >= 0 && per_traj >= 0, "philox_normal: bad argument");
    return launch_philox_normal(out, B, per_traj, seed, traj0, draw, (hipStream_t)stream);
}

size_t dpc_conv_workspace_bytes(int Cin, int Cout, int ntaps) {
    // room for the fp32 pack (128 B per (n, 32-channel chunk, tap)), the bf16x6 pack (192 B) or the Winograd F(4,3) pack of a 27-tap
    // convolution (54 x 128 B per (n, 32-channel chunk) = 256 B per tap)
    return (size_t)ntaps * igemm_kchunks(Cin) * igemm_npad(Cout) * 256 + 256;
}

int dpc_conv3d_cl(const float* x_cl, const float* w_ref, const float* bias, float* out_cl, int B, int F, int H, int W,
                  int Cin, int Cout, int kd, int kh, int kw, int sd, int sh, int sw, int pd, int ph, int pw, void* ws,
                  size_t ws_bytes, dpc_stream_t stream) {
    DPC_REQUIRE(x_cl && w_ref && out_cl && ws, "conv3d_cl: null argument");
    DPC_REQUIRE(sd == 1, "conv3d_cl: the frame axis is never strided (conv3d.py:159-163)");
    const int ntaps = kd * kh * kw;
    DPC_REQUIRE(ntaps >= 1 && ntaps <= 32, "conv3d_cl: 1..32 taps (the 7x7x7 stem has its own kernel)");
    DPC_REQUIRE(ws_bytes >= dpc_conv_workspace_bytes(Cin, Cout, ntaps), "conv3d_cl: workspace too small");
    hipStream_t s = (hipStream_t)stream;
    float* wp = reinterpret_cast<float*>(align_up((size_t)ws, 256));
    IgemmParams p{};
    int off[32];
    int t = 0;
    for (int a = 0; a < kd; ++a)
        for (int b = 0; b < kh; ++b)
            for (int c = 0; c < kw; ++c, ++t) {
                p.tdf[t] = (signed char)(a - pd);
                p.tdh[t] = (signed char)(b - ph);
                p.tdw[t] = (signed char)(c - pw);
                off[t] = t;
            }
    p.N = Cout; p.Npad = igemm_npad(Cout); p.kchunks = igemm_kchunks(Cin); p.ntaps = ntaps;
    if (kd == 3 && kh == 3 && kw == 3 && sh == 1 && sw == 1 && pd == 1 && ph == 1 && pw == 1) {
        // the U-Net's 3x3x3 convs run on the LDS halo-tile kernel (conv3h.hip)
        Conv3hParams q{};
        q.a0 = x_cl; q.C0 = Cin; q.wp = wp; q.bias = bias; q.out = out_cl;
        q.B = B; q.F = F; q.H = H; q.W = W; q.N = Cout; q.Npad = p.Npad; q.kchunks = (Cin + 15) / 16;
        if (conv_mode_default() == 2) {
            q.wpw = wp;                                 // (probe with the launcher's OWN predicate: the two must not diverge)
            const bool take_w = Cin % 32 == 0 && conv3w_supported(q);
            q.wpw = nullptr;
            if (take_w) {                               // Winograd pack: 36 x 64 B per (chunk, n)
                int rc = launch_pack_weights_w3(w_ref, wp, Cout, p.Npad, Cin, s);
                if (rc) return rc;
                q.wp = nullptr; q.wpw = wp;
                // perf attribution only (tools/bench_conv.py): DPC_CONV_FAKE_GN=1 times the fused GroupNorm+SiLU loader on a
                // constant coefficient table (y = x + 1); the result is then NOT the convolution of x
                static const int fake_gn = debug_switch("DPC_CONV_FAKE_GN", 0);
                if (fake_gn) {
                    static float* tab = nullptr;
                    static size_t cap = 0;
                    const size_t need = (size_t)B * Cin * 7 * sizeof(float);
                    if (need > cap) {
                        if (tab) (void)hipFree(tab);
                        DPC_HIP(hipMalloc(&tab, need));
                        cap = need;
                    }
                    DPC_HIP(hipMemsetD32Async(reinterpret_cast<hipDeviceptr_t>(tab), 0x3f800000, need / 4, s));
                    q.in_coef = tab;
                }
                return launch_conv3f3(q, s);
            }
            int rc = launch_pack_weights_f3(w_ref, wp, Cout, p.Npad, Cin, s);     // 64 B per (tap, chunk, n)
            if (rc) return rc;
            return launch_conv3f3(q, s);
        }
        if (conv_mode_default() == 1) {
            int rc = launch_pack_weights_x6(w_ref, wp, Cout, p.Npad, Cin, s);     // 96 B per (tap, chunk, n) <= fp32 pack size
            if (rc) return rc;
            return launch_conv3x6(q, s);
        }
        int rc = launch_pack_weights(w_ref, wp, Cout, p.Npad, Cin, 27, (long long)Cin * 27, 27, off, s, 16);
        if (rc) return rc;
        return launch_conv3h(q, s);
    }
    if (kd == 1 && kh == 3 && kw == 3 && sh == 1 && sw == 1 && pd == 0 && ph == 1 && pw == 1 && conv_mode_default() == 2 &&
        H % 8 == 0 && W % 8 == 0 && Cin % 4 == 0) {
        // (1,3,3): the big-tile halo kernel with the frames as independent images (the 2-D U-Net's 3x3 convs)
        Conv3hParams q{};
        q.a0 = x_cl; q.C0 = Cin; q.wp = wp; q.bias = bias; q.out = out_cl;
        q.B = 1; q.F = B * F; q.H = H; q.W = W; q.N = Cout; q.Npad = p.Npad; q.kchunks = (Cin + 15) / 16; q.kd = 1;
        int rc = launch_pack_weights_f3(w_ref, wp, Cout, p.Npad, Cin, s, 9);
        if (rc) return rc;
        return launch_conv3f3(q, s);
    }
    const bool x6 = igemm_mode_default() >= 1;
    int rc = x6 ? launch_pack_weights_g6(w_ref, wp, Cout, p.Npad, Cin, ntaps, (long long)Cin * ntaps, ntaps, off, s)
                : launch_pack_weights(w_ref, wp, Cout, p.Npad, Cin, ntaps, (long long)Cin * ntaps, ntaps, off, s);
    if (rc) return rc;
    const int Ho = (H + 2 * ph - kh) / sh + 1, Wo = (W + 2 * pw - kw) / sw + 1;
    p.a0 = x_cl; p.a1 = nullptr; p.C0 = Cin; p.C1 = 0; p.wp = wp; p.bias = bias; p.resid = nullptr; p.out = out_cl;
    p.BF = B * F; p.F = F; p.Hi = H; p.Wi = W; p.Ho = Ho; p.Wo = Wo; p.sh = sh; p.sw = sw;
    p.out_mode = 0;
    p.M = (long long)B * F * Ho * Wo;
    return x6 ? launch_igemm6(p, wp, s) : launch_igemm(p, s);
}

int dpc_convtranspose3d_144_cl(const float* x_cl, const float* w_ref, const float* bias, float* out_cl, int B, int F,
                               int H, int W, int Cin, int Cout, void* ws, size_t ws_bytes, dpc_stream_t stream) {
    DPC_REQUIRE(x_cl && w_ref && out_cl && ws, "convtranspose3d: null argument");
    DPC_REQUIRE(ws_bytes >= 4 * dpc_conv_workspace_bytes(Cin, Cout, 4), "convtranspose3d: workspace too small");
    hipStream_t s = (hipStream_t)stream;
    const size_t per = align_up(dpc_conv_workspace_bytes(Cin, Cout, 4), 256);
    const int dh_[2][2] = {{0, -1}, {1, 0}}, kh_[2][2] = {{1, 3}, {0, 2}};
    for (int a = 0; a < 2; ++a)
        for (int b = 0; b < 2; ++b) {
            float* wp = reinterpret_cast<float*>(align_up((size_t)ws, 256) + (size_t)(a * 2 + b) * per);
            IgemmParams p{};
            int off[32];
            int t = 0;
            for (int u = 0; u < 2; ++u)
                for (int v = 0; v < 2; ++v, ++t) {
                    p.tdf[t] = 0;
                    p.tdh[t] = (signed char)dh_[a][u];
                    p.tdw[t] = (signed char)dh_[b][v];
                    off[t] = kh_[a][u] * 4 + kh_[b][v];
                }
            p.N = Cout; p.Npad = igemm_npad(Cout); p.kchunks = igemm_kchunks(Cin); p.ntaps = 4;
            const bool x6 = igemm_mode_default() >= 1;
            int rc = x6 ? launch_pack_weights_g6(w_ref, wp, Cout, p.Npad, Cin, 4, 16, (long long)Cout * 16, off, s)
                        : launch_pack_weights(w_ref, wp, Cout, p.Npad, Cin, 4, 16, (long long)Cout * 16, off, s);
            if (rc) return rc;
            p.a0 = x_cl; p.C0 = Cin; p.wp = wp; p.bias = bias; p.out = out_cl;
            p.BF = B * F; p.F = F; p.Hi = H; p.Wi = W; p.Ho = H; p.Wo = W; p.sh = 1; p.sw = 1;
            p.out_mode = 2; p.par_a = a; p.par_b = b;
            p.M = (long long)B * F * H * W;
            rc = x6 ? launch_igemm6(p, wp, s) : launch_igemm(p, s);
            if (rc) return rc;
        }
    return DPC_OK;
}

size_t dpc_groupnorm_workspace_bytes(int B, int C) { return gn_workspace_bytes(B, C) + 256; }

int dpc_groupnorm_silu_cl(float* x_cl, const float* gamma, const float* beta, const float* scale_shift, int B,
                          int64_t rows_per_sample, int C, int groups, void* ws, size_t ws_bytes, dpc_stream_t stream) {
    DPC_REQUIRE(x_cl && gamma && beta && ws, "groupnorm_silu: null argument");
    DPC_REQUIRE(ws_bytes >= dpc_groupnorm_workspace_bytes(B, C), "groupnorm_silu: workspace too small");
    return launch_groupnorm_silu(x_cl, x_cl, nullptr, gamma, beta, scale_shift, B, rows_per_sample, C, groups,
                                 reinterpret_cast<void*>(align_up((size_t)ws, 256)), (hipStream_t)stream);
}

int dpc_attention_core(const float* qkv, float* out, int heads, int L, int64_t n_seq, int64_t seq_inner,
                       int64_t seq_outer_stride_rows, int64_t seq_inner_stride_rows, int64_t token_stride_rows,
                       const float* rot_cos, const float* rot_sin, const float* bias, dpc_stream_t stream) {
    DPC_REQUIRE(qkv && out && seq_inner >= 1, "attention_core: bad argument");
    AttnParams p{};
    p.qkv = qkv; p.out = out; p.heads = heads; p.L = L; p.n_seq = n_seq; p.seq_inner = seq_inner;
    p.seq_outer_stride = seq_outer_stride_rows; p.seq_inner_stride = seq_inner_stride_rows;
    p.token_stride = token_stride_rows; p.rot_cos = rot_cos; p.rot_sin = rot_sin; p.bias = bias;
    return launch_attention(p, (hipStream_t)stream);
}

size_t dpc_linear_attention_workspace_bytes(int64_t images, int heads) {
    return linattn_workspace_bytes(images, heads) + 256;
}

int dpc_linear_attention_core(const float* qkv, float* out, int heads, int64_t images, int N, void* ws, size_t ws_bytes,
                              dpc_stream_t stream) {
    DPC_REQUIRE(qkv && out && ws, "linear_attention_core: null argument");
    DPC_REQUIRE(ws_bytes >= dpc_linear_attention_workspace_bytes(images, heads), "linear_attention_core: workspace too small");
    return launch_linear_attention(qkv, out, heads, images, N, reinterpret_cast<void*>(align_up((size_t)ws, 256)),
                                   (hipStream_t)stream);
}

int dpc_burgers_fd(const float* u0, const float* f, float* traj, int N, int nx, int num_t, double visc, double T,
                   double dt, dpc_stream_t stream) {
    DPC_REQUIRE(u0 && f && traj && N >= 0, "burgers_fd: bad argument");
    return launch_burgers_fd(u0, f, traj, N, nx, num_t, visc, T, dt, (hipStream_t)stream);
}

}  // extern "C"
