"""Host side of diffphycon_amd.sequence and of the dpc_seq_* entries: sizes of scratch, and calls at the border of what is supported."""
import ctypes as C

import pytest
import torch

from diffphycon_amd import _lib, sequence as S


def _attn(**kw):
    a = _lib.SeqAttn(type=2, batch=1, heads=2, kv_heads=1, head_dim=32, q_len=4, k_len=4, scale=1.0, lse_rows=8, lse=256)
    for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        setattr(a, n, _lib.SeqTensor(4096, 256, 64, 32))
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def _padded(ql, kl, q_max, H, Hk, D, causal):
    """The dpc_seq_attn of a padded plan (addresses are not looked at)."""
    blocks = [len(S.SequencePlan._tiles(ql, kl, keys, causal)) for keys in (False, True)]
    return _attn(q_tiles=4096, k_tiles=4096, n_q_tiles=blocks[0], n_k_tiles=blocks[1], batch=len(ql), heads=H, kv_heads=Hk, head_dim=D, q_len=max(ql), k_len=max(kl),
                 causal=causal, lse_rows=len(ql) * H * q_max)


# ---------------------------------------------------------------------------------------------------------------- scratch
def test_scratch_of_a_padded_plan_goes_by_its_sequences_not_by_the_buffer():
    """Partial sums exist for the blocks of 128 rows that the sequences have, times the splits: at most 1024 x 128 rows in all, whatever the buffer's size."""
    need = lambda a, b: _lib.lib().dpc_seq_attn_workspace_bytes(C.byref(a), b)  # noqa: E731
    ql = [4096] + [64] * 63
    a = _padded(ql, ql, 4096, 1, 1, 128, 1)
    rows = 8 * a.lse_rows                                            # two floats a row of lse
    assert 0 < need(a, 1) <= rows + 1024 * 128 * 256 * 4 + 4096 and 0 < need(a, 0) <= 1024 * 128 * 130 * 4 + 4096
    ql = [1] * 8
    a = _padded(ql, [16384] * 8, 16384, 32, 8, 128, 0)               # one token a sequence in a long buffer: 4 rows a key head
    assert 0 < need(a, 0) <= 512 * 4 * 130 * 4 + 4096
    for D in (8, 64, 128):                                           # and of dense calls
        for B, Lq, Lk, H, Hk in ((1, 4096, 4096, 1, 1), (8, 1, 16384, 32, 8), (3, 333, 2501, 10, 5), (1, 7, 100000, 4, 4), (2, 50000, 300, 2, 1)):
            for causal in (0, 1):
                a = _attn(batch=B, heads=H, kv_heads=Hk, head_dim=D, q_len=Lq, k_len=Lk, causal=causal, lse_rows=B * H * Lq)
                assert need(a, 1) <= 8 * a.lse_rows + 1024 * 128 * 2 * D * 4 + 4096 and need(a, 0) <= 1024 * 128 * (D + 2) * 4 + 4096


# ---------------------------------------------------------------------------------------------------------------- strides
@pytest.mark.parametrize("es,dtype", [(2, torch.bfloat16), (4, torch.float32)])
def test_token_strides_are_copied_exactly_where_the_entry_refuses_them(es, dtype):
    """Around the largest token stride that a kernel reads (64 rows within 2^31 bytes): a layout that is not copied is one that the entry takes."""
    need = _lib.lib().dpc_seq_attn_workspace_bytes
    taken = set()
    for stride in range((1 << 25) - 160, (1 << 25) + 33, 16):
        x = torch.empty(stride // es + 8, dtype=dtype).as_strided((1, 2, 1, 8), (0, stride // es, 8, 1))
        as_is = S._lay(x, es)[0] is x
        assert as_is == S._ok16(x, es)
        a = _attn(type=0 if es == 4 else 2, head_dim=8, q=_lib.SeqTensor(4096, 0, stride // es, 8))
        entry = need(C.byref(a), 1) > 0
        assert as_is == entry, (stride, as_is, entry)
        if not entry:
            assert b"token strides" in _lib.lib().dpc_last_error()
        taken.add(entry)
    assert taken == {True, False}


# ---------------------------------------------------------------------------------------------------------------- sizes
@pytest.mark.parametrize("n", [(1 << 30) + 1, 1 << 31, (1 << 32) + 8])
def test_layer_norm_refuses_rows_beyond_its_range(n):
    """A width that the entry's 32 bits cannot hold is refused, not cut off; rows are at most 2^30 elements wide."""
    x = torch.zeros(1).expand(1, n)
    st = torch.zeros(1, 2)
    for f in (lambda: S.layer_norm_forward(x), lambda: S.layer_norm_backward(x, x, st), lambda: S.layer_norm_forward(x[:0]), lambda: S.layer_norm_backward(x[:0], x[:0], st[:0])):
        with pytest.raises(ValueError, match="2\\^30"):
            f()


def test_layer_norm_entries_refuse_rows_beyond_their_range():
    L, p = _lib.lib(), C.c_void_p(4096)
    assert L.dpc_seq_norm_fwd(p, None, None, p, p, 1, (1 << 30) + 1, 1 << 31, 1e-5, 0, 0, None) < 0 and b"C" in L.dpc_last_error()
    need = L.dpc_seq_norm_bwd_workspace_bytes(1, 1 << 30, 0)
    assert need >= 2 * (1 << 30) * 4 and L.dpc_seq_norm_bwd_workspace_bytes(1, (1 << 30) + 1, 0) == 0
    assert L.dpc_seq_norm_bwd(p, p, p, None, p, p, p, 1, (1 << 30) + 1, 1 << 31, 1 << 31, 0, 0, p, 1 << 40, None) < 0


def test_attention_and_rotary_refuse_sizes_beyond_32_bits_in_their_own_manner():
    """Broadcast tensors of 2^31 rows cost nothing to make: ValueError, not the packing's own error (nor RuntimeError: shapes come before devices)."""
    z, far = torch.zeros(1, 1, 1, 8), 1 << 31
    many, long, wide = z.expand(far, 1, 1, 8), z.expand(1, far, 1, 8), z.expand(1, 1, far, 8)
    for q, k in ((many, many), (long, z), (z, long), (wide, z), (long, long)):
        with pytest.raises(ValueError, match="2\\^31"):
            S.attention_forward(q, k, k)
        with pytest.raises(ValueError, match="2\\^31"):
            S.attention_backward(q, q, k, k, q, torch.zeros(1, 1, 1))
    table = type("T", (), dict(table=torch.zeros(16, 4, 2), rotary_dim=8, max_positions=1 << 40, layout="half", stream=None))
    for q in (many, long, wide, torch.zeros(1, 1, 1, 1).expand(1, 1, 1, far)):
        for k in (q, None):
            with pytest.raises(ValueError, match="2\\^31"):
                S.rotary_forward(q, k, table)


def test_entries_refuse_launches_of_more_threads_than_32_bits_count():
    """Before anything is launched: 2^24 workgroups of 256 threads are one launch too many."""
    L = _lib.lib()
    a = _attn(batch=1 << 24, heads=1, lse_rows=1 << 26)
    ws = C.c_void_p(1 << 20)
    for rc in (L.dpc_seq_attn_fwd(C.byref(a), ws, 1 << 40, None), L.dpc_seq_attn_bwd(C.byref(a), ws, 1 << 40, None)):
        assert rc < 0 and b"grid too large" in L.dpc_last_error()
    T = _lib.SeqTensor(4096, 0, 64 * 128, 128)
    for interleaved in (0, 1):
        a = _lib.SeqRotary(xq=T, yq=_lib.SeqTensor(8192, 0, 64 * 128, 128), table=4096, max_positions=1 << 30, type=0, batch=1, tokens=1 << 25, heads=64, head_dim=128, rotary_dim=128,
                           interleaved=interleaved)
        assert L.dpc_seq_rotary_run(C.byref(a), None) < 0 and b"grid too large" in L.dpc_last_error()


# ---------------------------------------------------------------------------------------------------------------- buffers that overlap
def _elements(x):
    at = torch.tensor([x.storage_offset()])
    for n, s in zip(x.shape, x.stride()):
        at = (at[:, None] + torch.arange(n) * s).flatten()
    return set(at.tolist())


def test_overlap_finds_every_shared_element():
    """Pairs of views of one storage with equal outer strides, batches that are no whole number of tokens apart among them: never "apart" where an element is
    shared; and views of one projection, padded or not, are apart."""
    base, g = torch.zeros(4000), torch.Generator().manual_seed(2)
    r = lambda lo, hi: int(torch.randint(lo, hi, (1,), generator=g))  # noqa: E731
    apart = 0
    for _ in range(4000):
        outer = (r(1, 60), r(1, 60))
        sizes = (r(1, 4), r(1, 4), r(1, 4), r(1, 5))
        a, b = (base.as_strided(sizes, (*outer, r(1, 9), 1), r(0, 40)) for _ in range(2))
        shared = bool(_elements(a) & _elements(b))
        found = S._overlap(a, b)
        assert found or not shared, (a.shape, a.stride(), a.storage_offset(), b.stride(), b.storage_offset())
        apart += not found
    assert apart > 500
    a = base.as_strided((2, 2, 1, 3), (10, 7, 3, 1))                 # rows at 0, 7, 10, 17; the other's at 3, 10, 13, 20
    assert S._overlap(a, base.as_strided((2, 2, 1, 3), (10, 7, 3, 1), 3))
    for stride_b in (5 * 96, 5 * 96 + 17):
        q, k, v = (base.as_strided((2, 5, 4, 8), (stride_b, 96, 8, 1), 32 * i) for i in range(3))
        assert not S._overlap(q, k) and not S._overlap(k, v) and not S._overlap(q, v)


def test_rotary_refuses_buffers_whose_own_elements_overlap():
    """In place or not: two threads would write one element.  Views of a projection and of a buffer with gaps are fine."""
    base = torch.zeros(4096)
    q = torch.zeros(2, 4, 3, 8)
    fine = [torch.zeros_like(q), torch.zeros(2, 4, 5, 8)[:, :, 1:4], base.as_strided((2, 4, 3, 8), (8, 16, 64, 1)), torch.zeros(3, 4, 2, 8).transpose(0, 2)]
    for y in fine:
        assert S._rotary_out(q, None, (y,))[0] is y
    for y in (base.as_strided((2, 4, 3, 8), (96, 16, 8, 1)), base.as_strided((2, 4, 3, 8), (96, 24, 4, 1)), base.as_strided((2, 4, 3, 8), (40, 24, 8, 1)), q[:, :1].expand_as(q)):
        with pytest.raises(ValueError):
            S._rotary_out(q, None, (y,))
    x = base.as_strided((1, 4, 3, 8), (96, 16, 8, 1))                # in place on an input that overlaps itself
    with pytest.raises(ValueError):
        S._rotary_out(x, None, (x,))


@pytest.mark.parametrize("kw", [dict(trained_positions=float("nan")), dict(trained_positions=0), dict(trained_positions=-5.0),
                                dict(turns=(1.0, float("nan")))])
def test_rotary_table_refuses_a_ramp_without_meaning(kw):
    with pytest.raises(ValueError):
        S.RotaryTable(8, 16, scaling="ramp", factor=2.0, **kw)


@pytest.mark.parametrize("scale", [1e39, 3.5e38, 1e-60, 1e-39])
def test_attention_refuses_scales_beyond_fp32(scale):
    """A scale that 32 bits make 0 or infinity is refused as one that is 0 or infinity is."""
    q = torch.zeros(1, 2, 1, 8)
    with pytest.raises(ValueError, match="scale"):
        S.attention_forward(q, q, q, scale=scale)
    with pytest.raises(ValueError, match="scale"):
        S.attention_backward(q, q, q, q, q, torch.zeros(1, 1, 2), scale=scale)


def test_attention_entries_refuse_key_axes_whose_splits_would_pass_32_bits():
    """Splits are whole tiles, up to 512 of them: the last one ends up to 2^16 behind the last key, and that has to be a 32-bit number too."""
    L = _lib.lib()
    for k_len, fine in (((1 << 31) - (1 << 17), True), ((1 << 31) - (1 << 17) + 1, False), ((1 << 31) - 300, False), ((1 << 31) - 257, False)):
        for q_len in (1, 40):
            a = _attn(q_len=q_len, k_len=k_len)
            assert (L.dpc_seq_attn_workspace_bytes(C.byref(a), 0) > 0) == fine, (q_len, k_len)
            if not fine:
                assert L.dpc_seq_attn_fwd(C.byref(a), C.c_void_p(4096), 1 << 40, None) < 0 and b"too long" in L.dpc_last_error()
