"""diffphycon_amd.sequence and the dpc_seq_* entries refuse what they cannot compute, on the host, before anything is launched."""
import ctypes as C
import types

import pytest
import torch

from diffphycon_amd import _lib, sequence as S


def _qkv(B=2, Lq=4, Lk=6, H=4, Hk=2, D=16, dtype=torch.float32):
    return torch.zeros(B, Lq, H, D, dtype=dtype), torch.zeros(B, Lk, Hk, D, dtype=dtype), torch.zeros(B, Lk, Hk, D, dtype=dtype)


@pytest.mark.parametrize("change,error", [
    (dict(), RuntimeError),                                          # CPU tensors: there is no CPU path
    (dict(dtype=torch.float64), TypeError),
    (dict(D=12), ValueError), (dict(D=136), ValueError),
    (dict(H=3), ValueError),                                         # not a multiple of the key heads
    (dict(scale=0.0), ValueError), (dict(scale=-1.0), ValueError), (dict(scale=float("nan")), ValueError),
    (dict(mask=torch.ones(2, 5, dtype=torch.bool)), ValueError),
    (dict(mask=torch.ones(2, 6, dtype=torch.uint8)), ValueError),
])
def test_attention_refuses(change, error):
    kw = dict(change)
    scale, mask = kw.pop("scale", None), kw.pop("mask", None)
    q, k, v = _qkv(**kw)
    with pytest.raises(error):
        S.attention_forward(q, k, v, scale=scale, key_mask=mask)
    with pytest.raises(error):
        S.attention_backward(q, q, k, v, q, torch.zeros(q.shape[0], q.shape[2], q.shape[1]), scale=scale, key_mask=mask)


def test_attention_refuses_shapes_and_types_that_disagree():
    q, k, v = _qkv()
    with pytest.raises(ValueError):
        S.attention_forward(q, k, v[:, :5])
    with pytest.raises(ValueError):
        S.attention_forward(q[:1], k, v)
    with pytest.raises(ValueError):
        S.attention_forward(q[0], k[0], v[0])                         # packed layout without a plan
    with pytest.raises(ValueError):
        S.attention_forward(q, k[..., :8], v[..., :8])
    with pytest.raises(TypeError):
        S.attention_forward(q, k.half(), v)
    with pytest.raises(ValueError):
        S.attention_backward(q[:, :3], q, k, v, q, torch.zeros(2, 4, 4))
    with pytest.raises(ValueError):
        S.attention_backward(q, q, k, v, q[:, :3], torch.zeros(2, 4, 4))


@pytest.mark.parametrize("args,kw", [
    (([], []), {}), (([3], [3, 4]), {}), (([3, -1],), {}), (([1 << 30, 1 << 30, 1 << 30],), {}),
])
def test_plan_refuses(args, kw):
    with pytest.raises(ValueError):
        S.SequencePlan.packed(*args, **kw)


def test_plan_refuses_lengths_beyond_the_padding_and_the_cpu():
    with pytest.raises(ValueError):
        S.SequencePlan.padded([3, 5], 4)
    with pytest.raises(ValueError):
        S.SequencePlan.padded([3, 4], 4, [9, 1], 8)
    with pytest.raises(RuntimeError):
        S.SequencePlan.packed([3, 4], device="cpu")


def test_plan_lists_every_block_once_most_work_first():
    ql, kl = [0, 300, 1, 128, 700], [5, 300, 1, 400, 600]
    for causal in (False, True):
        q = S.SequencePlan._tiles(ql, kl, False, causal)
        k = S.SequencePlan._tiles(ql, kl, True, causal)
        assert sorted(q) == [(b, t) for b in range(5) for t in range((ql[b] + 127) // 128)]
        assert sorted(k) == [(b, t) for b in range(5) for t in range((kl[b] + 127) // 128)]
        assert q[0][0] == k[0][0] == 4 and q[-1] == (2, 0)
    assert S.SequencePlan._tiles(ql, kl, False, True)[0] == (4, 5) and S.SequencePlan._tiles(ql, kl, True, True)[0] == (4, 0)
    assert S.SequencePlan._tiles([0], [0], False, True) == []


@pytest.mark.parametrize("kw", [
    dict(rotary_dim=7), dict(rotary_dim=0), dict(max_positions=0), dict(layout="other"), dict(scaling="other"), dict(factor=2.0),
    dict(scaling="linear", factor=0.5), dict(scaling="ntk", factor=2.0, rotary_dim=2), dict(scaling="ramp", factor=2.0, turns=(3.0, 3.0)),
    dict(base=0.0), dict(base=float("inf")),
])
def test_rotary_table_refuses(kw):
    kw = dict(dict(rotary_dim=8, max_positions=16), **kw)
    with pytest.raises(ValueError):
        S.RotaryTable(kw.pop("rotary_dim"), kw.pop("max_positions"), **kw)


def test_rotary_refuses():
    table = types.SimpleNamespace(table=torch.zeros(16, 4, 2), rotary_dim=8, max_positions=16, layout="half", stream=None)
    q, k = torch.zeros(2, 4, 3, 16), torch.zeros(2, 4, 1, 16)
    ok = torch.zeros(4, dtype=torch.int64)
    for error, args, kw in [
        (RuntimeError, (q, k), {}), (ValueError, (q[0, 0], None), {}), (ValueError, (q, k[:, :3]), {}), (ValueError, (q, k[..., :8]), {}),
        (TypeError, (q, k.half()), {}), (TypeError, (q.double(), None), {}), (ValueError, (q[..., :4], None), {}),
        (ValueError, (q, k), dict(start=13)), (ValueError, (q, k), dict(start=-1)), (ValueError, (q, k), dict(positions=ok, start=1)),
        (TypeError, (q, k), dict(positions=ok.float())), (ValueError, (q, k), dict(positions=ok[:3])), (ValueError, (q[0], k[0]), dict(positions=torch.zeros(1, 4).long())),
    ]:
        for f in (S.rotary_forward, S.rotary_backward):
            with pytest.raises(error):
                f(*args, table, **kw)


def test_layer_norm_refuses():
    x, w = torch.zeros(3, 8), torch.ones(8)
    st = torch.zeros(3, 2)
    for error, f in [
        (RuntimeError, lambda: S.layer_norm_forward(x, w)), (TypeError, lambda: S.layer_norm_forward(x.double())),
        (ValueError, lambda: S.layer_norm_forward(x, w[:7])), (TypeError, lambda: S.layer_norm_forward(x, w.half())),
        (TypeError, lambda: S.layer_norm_forward(x.half(), w, w.half())), (ValueError, lambda: S.layer_norm_forward(x, eps=0.0)),
        (ValueError, lambda: S.layer_norm_forward(torch.zeros(3, 0))), (ValueError, lambda: S.layer_norm_forward(torch.zeros(()))),
        (RuntimeError, lambda: S.layer_norm_backward(x, x, st, w)), (ValueError, lambda: S.layer_norm_backward(x[:2], x, st, w)),
        (ValueError, lambda: S.layer_norm_backward(x, x, st[:2], w)), (TypeError, lambda: S.layer_norm_backward(x, x.half(), st, w)),
        (TypeError, lambda: S.layer_norm_backward(x, x, st, w, param_dtype=torch.float16)),
    ]:
        with pytest.raises(error):
            f()


def test_overlap_of_views():
    a = torch.zeros(2, 5, 3, 4, 8)
    q, k, v = a.unbind(2)
    assert not S._overlap(q, k) and not S._overlap(k, v) and S._overlap(q, q)
    assert S._overlap(a[:, :, 0], a[:, :, :2].flatten(2, 3)) and not S._overlap(q, torch.zeros(2))
    b = torch.zeros(64)
    assert S._overlap(b[:40], b[32:]) and not S._overlap(b[:32], b[32:])


def _attn(**kw):
    a = _lib.SeqAttn(type=2, batch=1, heads=2, kv_heads=1, head_dim=32, q_len=4, k_len=4, scale=1.0, lse_rows=8, lse=256)
    for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        setattr(a, n, _lib.SeqTensor(4096, 256, 64, 32))
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw", [
    dict(type=3), dict(batch=-1), dict(q_len=-1), dict(heads=3, kv_heads=2), dict(kv_heads=0), dict(head_dim=36), dict(head_dim=0), dict(head_dim=256),
    dict(scale=0.0), dict(scale=float("inf")), dict(q=_lib.SeqTensor(None, 0, 0, 0)), dict(k=_lib.SeqTensor(4100, 256, 64, 32)),
    dict(v=_lib.SeqTensor(4096, 256, 63, 32)), dict(lse=None), dict(q_tiles=4096, n_q_tiles=1), dict(n_q_tiles=1), dict(q_tiles=4112, k_tiles=4096, n_q_tiles=1),
])
def test_attention_entries_refuse(kw):
    L = _lib.lib()
    a = _attn(**kw)
    for rc in (L.dpc_seq_attn_fwd(C.byref(a), None, 0, None), L.dpc_seq_attn_bwd(C.byref(a), C.c_void_p(4096), 1 << 20, None)):
        assert rc < 0 and b"seq_attn" in L.dpc_last_error()


def test_attention_backward_entry_refuses_a_small_workspace():
    L = _lib.lib()
    a = _attn()
    need = L.dpc_seq_attn_workspace_bytes(C.byref(a), 1)
    assert need >= 2 * 8 * 4
    assert L.dpc_seq_attn_bwd(C.byref(a), C.c_void_p(4096), need - 1, None) < 0
    assert L.dpc_seq_attn_bwd(C.byref(a), None, need, None) < 0
    assert L.dpc_seq_attn_fwd(None, None, 0, None) < 0


def test_rotary_and_norm_entries_refuse():
    L = _lib.lib()
    p = C.c_void_p(4096)
    T = _lib.SeqTensor(4096, 256, 64, 32)
    ok = dict(xq=T, yq=T, table=4096, max_positions=4, type=0, batch=1, tokens=4, heads=2, kv_heads=0, head_dim=32, rotary_dim=32)
    for kw in (dict(type=-1), dict(rotary_dim=31), dict(rotary_dim=64), dict(rotary_dim=0), dict(table=None), dict(heads=0), dict(xk=T), dict(batch=-1),
               dict(batch=1 << 16, tokens=1 << 16), dict(max_positions=0)):
        a = _lib.SeqRotary(**dict(ok, **kw))
        assert L.dpc_seq_rotary_run(C.byref(a), None) < 0, kw
    assert L.dpc_seq_rotary_run(None, None) < 0
    for args in [(None, None, None, p, p, 4, 8, 8, 1e-5, 0, 0), (p, None, None, p, p, 4, 0, 8, 1e-5, 0, 0), (p, None, None, p, p, 4, 8, 7, 1e-5, 0, 0),
                 (p, None, None, p, p, 4, 8, 8, 0.0, 0, 0), (p, None, None, p, p, 4, 8, 8, 1e-5, 3, 0), (p, None, None, p, p, 4, 8, 8, 1e-5, 1, 2)]:
        assert L.dpc_seq_norm_fwd(*args, None) < 0
    need = L.dpc_seq_norm_bwd_workspace_bytes(400, 800, 0)
    assert need >= 2 * 800 * 4
    assert L.dpc_seq_norm_bwd(p, p, p, None, p, p, p, 400, 800, 800, 800, 0, 0, p, need - 1, None) < 0
    assert L.dpc_seq_norm_bwd(p, p, p, None, p, p, p, 0, 800, 800, 800, 0, 0, p, need, None) < 0
