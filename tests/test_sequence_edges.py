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
