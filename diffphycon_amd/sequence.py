"""Operators on token sequences: layer norm, rotary positions and attention, forward and backward, on libdpc (include/dpc.h: dpc_seq_*).

As everywhere in this package the backward passes are explicit calls on the tensors the forward left, not an autograd graph: a training
step calls `*_forward`, keeps what it returns, and calls `*_backward`.  A pre-norm attention block is

    y, stats = layer_norm_forward(x, w, b)
    q, k = rotary_forward(q, k, table)                       # q, k, v: the caller's projections of y
    out, lse = attention_forward(q, k, v, causal=True)
    dq, dk, dv = attention_backward(dout, q, k, v, out, lse, causal=True)
    dq, dk = rotary_backward(dq, dk, table)
    dx, dw, db = layer_norm_backward(dy, x, stats, w)

Element types: float32, float16, bfloat16 (one type per call); sums, statistics and norms are float32 whatever the type.  Kernels run on the
current stream of the tensors' device and never synchronise; outputs and scratch come from torch's allocator on that stream, so calls may be
captured into graphs (a graph that reads a RotaryTable or a SequencePlan needs it alive for as long as it is replayed).  Nothing is accumulated
with atomics: results repeat bit for bit.  Arguments are checked on the host (ValueError / TypeError / RuntimeError); tensors must live on the
GPU (no CPU path)."""
import math

import torch

from . import _lib

_TYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_BYTES = {torch.float32: 4, torch.float16: 2, torch.bfloat16: 2}
_FAR = ((1 << 31) - 4096) // 64                                      # bytes between tokens at most: 64 rows of a tile within 2^31 bytes (seq_attn.hip: MAX_TOKEN_STRIDE)


# ------------------------------------------------------------------------------------------------------------------ checks
def _type(x, *more):
    t = x.dtype
    if t not in _TYPE:
        raise TypeError(f"element type {t}: float32, float16 and bfloat16 are supported")
    for y in more:
        if y.dtype != t:
            raise TypeError(f"one element type per call, got {t} and {y.dtype}")
    return t


def _device(x, *more):
    """The index of the device that all tensors (None: absent) are on."""
    d = x.get_device()
    if d < 0:
        raise RuntimeError("libdpc needs device tensors (there is no CPU implementation)")
    for y in more:
        if y is not None and y.get_device() != d:
            raise RuntimeError(f"tensors on {x.device} and {y.device}")
    return d


def _elsewhere(x):
    """Whether x is on a GPU that is not the current one: the public functions then call themselves there."""
    d = x.get_device()
    return d >= 0 and d != torch.cuda.current_device()


def _stream(d):
    return torch._C._cuda_getCurrentRawStream(d)


def _in_use(owner, d):
    """The owner's table is read on the current stream: its memory is not handed on before that stream is done with it."""
    if _stream(d) != owner.stream:
        owner.table.record_stream(torch.cuda.current_stream(d))


class _Tables:
    """An owner of a device tensor `table` that is whole for whatever stream uses it; copies (copy.deepcopy, pickle) own and address their own."""

    def _settle(self):
        if self.table.is_cuda:
            torch.cuda.current_stream(self.table.device).synchronize()
            self.stream = _stream(self.table.get_device())

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._settle()


def _ok16(x, es):
    """Whether a kernel can read x as it lies: last axis contiguous, base and strides on 16 bytes, tokens at most _FAR bytes apart."""
    s = [n if m > 1 else 0 for n, m in zip(x.stride()[:-1], x.shape[:-1])]
    return x.stride(-1) == 1 and not any(n * es & 15 for n in s) and x.data_ptr() & 15 == 0 and s[-2] * es <= _FAR


def _lay(x, es):
    """(x or a contiguous copy that a kernel can read; its address, strides of batch, token, head) for [B, T, H, D] or packed [T, H, D]."""
    if x.dim() == 4:
        b, t, h, d = x.stride()
    else:
        b = 0
        t, h, d = x.stride()
    p = x.data_ptr()
    if d == 1 and not (p | b * es | t * es | h * es) & 15 and t * es <= _FAR:
        return x, p, b, t, h
    if x.numel() and not _ok16(x, es):
        x = x.clone(memory_format=torch.contiguous_format)
    return x, x.data_ptr(), *_strides(x)


def _strides(x):
    """Strides of batch, token, head; 0 for an axis of one element, whose stride means nothing."""
    s = [n if m > 1 else 0 for n, m in zip(x.stride()[:-1], x.shape[:-1])]
    return s if len(s) == 3 else [0] + s


def _shares(a, b):
    return a.untyped_storage().data_ptr() == b.untyped_storage().data_ptr()


def _overlap(a, b):
    """Whether a and b may share an element: equal strides and a shift that fits into a row of the two inner axes, and into every step of the
    outer ones, keep views of one projection apart."""
    if not (a.numel() and b.numel()) or not _shares(a, b):
        return False
    if a.dim() == b.dim() and a.dim() >= 2 and a.stride()[:-2] == b.stride()[:-2]:
        wide = lambda t: (t.shape[-2] - 1) * t.stride(-2) + (t.shape[-1] - 1) * t.stride(-1) + 1
        (lo, wl), (hi, wh) = sorted(((a.storage_offset(), wide(a)), (b.storage_offset(), wide(b))))
        reach, apart = hi - lo + wh, hi - lo >= wl
        for s, n in sorted(zip(a.stride()[:-2], map(max, a.shape, b.shape))):
            if n > 1:
                apart, reach = apart and s >= reach, reach + s * (n - 1)
        if apart:
            return False
    last = lambda t: t.storage_offset() + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return a.storage_offset() <= last(b) and b.storage_offset() <= last(a)


def _distinct(x):
    """Whether every element of x has a place of its own: each axis steps over all that the smaller strides reach."""
    reach = 0
    for s, n in sorted((s, n) for s, n in zip(x.stride(), x.shape) if n > 1):
        if s <= reach:
            return False
        reach += s * (n - 1)
    return True


def _written(x, like, name, inputs):
    """Checks a caller's output buffer: shape, type, layout of distinct elements, and no element shared with an input."""
    if x.shape != like.shape or x.dtype != like.dtype:
        raise ValueError(f"{name}: expected shape {tuple(like.shape)} of {like.dtype}, got {tuple(x.shape)} of {x.dtype}")
    if x.numel() and not _distinct(x):
        raise ValueError(f"{name}: elements of the buffer overlap")
    if x.numel() and not _ok16(x, x.element_size()):
        raise ValueError(f"{name}: the last axis must be contiguous, base and strides multiples of 16 bytes")
    if any(_overlap(x, i) for i in inputs):
        raise ValueError(f"{name}: the buffer overlaps an input")


# ------------------------------------------------------------------------------------------------------------------ layer norm
def _norm_params(x, weight, bias):
    """The type of weight and bias."""
    t = None
    for p in (weight, bias):
        if p is None:
            continue
        if p.shape != x.shape[-1:]:
            raise ValueError(f"weight, bias: expected shape {tuple(x.shape[-1:])}, got {tuple(p.shape)}")
        if p.dtype not in (torch.float32, x.dtype) or t not in (None, p.dtype):
            raise TypeError(f"weight, bias: both float32 or both {x.dtype}, got {p.dtype}")
        t = p.dtype
    return 0 if t is None else _TYPE[t]


def _matrix(x, n):
    """(x as [rows, n] with one row stride: a view where the layout allows it, else a copy; its row stride).  Broadcast rows are copied."""
    if x.dim() == 2:
        r, c = x.stride()
        if (c == 1 or n == 1) and (r >= n or x.shape[0] == 1):
            return x, max(r, n)
    y = x.reshape(-1, n)
    if (y.stride(1) != 1 and n > 1) or (y.shape[0] > 1 and y.stride(0) < n):
        y = y.clone(memory_format=torch.contiguous_format)
    return y, max(y.stride(0), n)


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5):
    """y = (x - mean) / sqrt(variance + eps) * weight + bias over the last axis (biased variance) -> (y, stats).

    x: any shape [..., C], C from 1 to 2^30, any strides; weight, bias: [C] of float32 or of x's type, or None.  stats [rows, 2] float32 = (mean,
    1 / sqrt(variance + eps)) is what `layer_norm_backward` needs."""
    if _elsewhere(x):
        with torch.cuda.device(x.device):
            return layer_norm_forward(x, weight, bias, eps)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 1 << 30:
        raise ValueError("x: at least one axis, the last one of 1 to 2^30 elements")
    if not 0 < eps < math.inf:
        raise ValueError("eps must be positive and finite")
    t = _TYPE[_type(x)]
    wt = _norm_params(x, weight, bias)
    d = _device(x, weight, bias)
    n = x.shape[-1]
    rows = x.numel() // n
    y = x.new_empty(x.shape)
    stats = x.new_empty((rows, 2), dtype=torch.float32)
    if rows == 0:
        return y, stats
    m, stride = _matrix(x, n)
    w = None if weight is None else weight.contiguous()
    b = None if bias is None else bias.contiguous()
    _lib.check(_lib.lib().dpc_seq_norm_fwd(m.data_ptr(), None if w is None else w.data_ptr(), None if b is None else b.data_ptr(), y.data_ptr(),
                                           stats.data_ptr(), rows, n, stride, eps, t, wt, _stream(d)))
    return y, stats


def layer_norm_backward(dy, x, stats, weight=None, param_grads=True, param_dtype=None):
    """Gradients of `layer_norm_forward` -> (dx, dweight, dbias): dx in x's shape, dweight and dbias [C] in weight's type (without a weight:
    `param_dtype`, float32 by default).  param_grads=False skips the two sums (None, None)."""
    if _elsewhere(x):
        with torch.cuda.device(x.device):
            return layer_norm_backward(dy, x, stats, weight, param_grads, param_dtype)
    if dy.shape != x.shape:
        raise ValueError(f"dy {tuple(dy.shape)} must have x's shape {tuple(x.shape)}")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 1 << 30:
        raise ValueError("x: at least one axis, the last one of 1 to 2^30 elements")
    t = _TYPE[_type(x, dy)]
    _norm_params(x, weight, None)
    n = x.shape[-1]
    rows = x.numel() // n
    if stats.shape != (rows, 2) or stats.dtype != torch.float32 or not stats.is_contiguous():
        raise ValueError(f"stats: the contiguous float32 [{rows}, 2] of layer_norm_forward, got {tuple(stats.shape)} of {stats.dtype}")
    pt = weight.dtype if weight is not None else param_dtype or torch.float32
    if pt not in (torch.float32, x.dtype) or (weight is not None and param_dtype not in (None, pt)):
        raise TypeError(f"param_dtype: float32 or {x.dtype}; with a weight, the weight's type")
    d = _device(x, dy, stats, weight)
    dx = x.new_empty(x.shape)
    dw, db = (x.new_empty(n, dtype=pt), x.new_empty(n, dtype=pt)) if param_grads else (None, None)
    if rows == 0:
        return dx, dw.zero_() if dw is not None else None, db.zero_() if db is not None else None
    L = _lib.lib()
    (mx, sx), (mdy, sdy) = _matrix(x, n), _matrix(dy, n)
    w = None if weight is None else weight.contiguous()
    nbytes = L.dpc_seq_norm_bwd_workspace_bytes(rows, n, t) if param_grads else 0
    ws = x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _lib.check(L.dpc_seq_norm_bwd(mdy.data_ptr(), mx.data_ptr(), stats.data_ptr(), None if w is None else w.data_ptr(), dx.data_ptr(),
                                  dw.data_ptr() if param_grads else None, db.data_ptr() if param_grads else None, rows, n, sdy, sx, t, _TYPE[pt],
                                  ws.data_ptr() if nbytes else None, nbytes, _stream(d)))
    return dx, dw, db


# ------------------------------------------------------------------------------------------------------------------ rotary positions
class RotaryTable(_Tables):
    """Cosines and sines of the rotary angles for positions 0 .. max_positions - 1 (computed in 64 bits, kept in float32 on the device).

    Pair i < rotary_dim / 2 turns by position * f_i with f_i = base^(-2 i / rotary_dim); `layout` says which elements are a pair:
    "interleaved" (2i, 2i + 1) or "half" (i, i + rotary_dim / 2).  `scaling` by `factor` >= 1 for contexts longer than the trained ones:
      None      as is;
      "linear"  f_i / factor;
      "ntk"     base * factor^(rotary_dim / (rotary_dim - 2)) in place of base: the slowest pair slows by factor, the fastest not at all;
      "ramp"    by how often a pair turns within `trained_positions` (default max_positions / factor): fewer than turns[0] times: f_i / factor,
                more than turns[1] times: f_i, in between the mixture linear in that count; cosines and sines times 0.1 ln(factor) + 1."""

    def __init__(self, rotary_dim, max_positions, *, base=10000.0, layout="interleaved", scaling=None, factor=1.0, trained_positions=None,
                 turns=(1.0, 32.0), device="cuda"):
        rotary_dim, max_positions, base, factor = int(rotary_dim), int(max_positions), float(base), float(factor)
        if rotary_dim < 2 or rotary_dim % 2:
            raise ValueError("rotary_dim must be even and at least 2")
        if max_positions < 1:
            raise ValueError("max_positions must be at least 1")
        if not (base > 0 and math.isfinite(base)):
            raise ValueError("base must be positive and finite")
        if layout not in ("interleaved", "half"):
            raise ValueError("layout: 'interleaved' | 'half'")
        if scaling not in (None, "linear", "ntk", "ramp"):
            raise ValueError("scaling: None | 'linear' | 'ntk' | 'ramp'")
        if not (factor >= 1 and math.isfinite(factor)) or (scaling is None and factor != 1):
            raise ValueError("factor must be finite and at least 1 (and needs a scaling)")
        if scaling == "ntk" and rotary_dim < 4:
            raise ValueError("scaling 'ntk' needs rotary_dim >= 4")
        if scaling == "ramp" and not (len(turns) == 2 and 0 <= turns[0] < turns[1]):
            raise ValueError("turns: two rising numbers")
        if scaling == "ramp" and trained_positions is not None and not float(trained_positions) > 0:
            raise ValueError("trained_positions must be positive")
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("libdpc needs device tensors (there is no CPU implementation)")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a RotaryTable is computed and waited for: build it before the capture")
        exponent = -torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim
        f = (base * factor ** (rotary_dim / (rotary_dim - 2)) if scaling == "ntk" else base) ** exponent
        self.attention_factor = 1.0
        if scaling == "linear":
            f = f / factor
        elif scaling == "ramp":
            count = (max_positions / factor if trained_positions is None else float(trained_positions)) * f / (2 * math.pi)
            keep = ((count - turns[0]) / (turns[1] - turns[0])).clamp(0.0, 1.0)
            f = f / factor * (1 - keep) + f * keep
            self.attention_factor = 0.1 * math.log(factor) + 1.0
        self.rotary_dim, self.max_positions, self.layout, self.frequencies = rotary_dim, max_positions, layout, f
        angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * f.to(device)
        z = torch.polar(torch.full((), self.attention_factor, dtype=torch.float64, device=device), angle)
        self.table = torch.view_as_real(z).float().contiguous()                        # [max_positions, rotary_dim / 2, 2]
        self.interleaved = layout == "interleaved"
        self._settle()


def _rotary(q, k, table, positions, start, out, transpose):
    if _elsewhere(q):
        with torch.cuda.device(q.device):
            return _rotary(q, k, table, positions, start, out, transpose)
    packed, start = q.dim() == 3, int(start)
    if not packed and q.dim() != 4:
        raise ValueError("expected [batch, tokens, heads, head_dim] or packed [tokens, heads, head_dim]")
    t = _TYPE[_type(q) if k is None else _type(q, k)]
    shape = q.shape
    B, T, H, D = (1, *shape) if packed else shape
    Hk = 0
    if k is not None:
        ks = k.shape
        if len(ks) != len(shape) or (1, *ks)[-4] != B or ks[-3] != T or ks[-1] != D:
            raise ValueError(f"q {tuple(shape)} and k {tuple(ks)} must agree but for the heads")
        Hk = ks[-2]
    if H < 1 or (k is not None and Hk < 1):
        raise ValueError("at least one head")
    if (B | T | H | Hk | D) >> 31:
        raise ValueError(f"q {tuple(shape)}: axes of 2^31 or more are not supported")
    if table.rotary_dim > D:
        raise ValueError(f"the table's rotary_dim {table.rotary_dim} exceeds the head's {D}")
    pos_b = 0
    if positions is not None:
        if start != 0:
            raise ValueError("give positions or start, not both")
        if positions.dtype not in (torch.int64, torch.int32):
            raise TypeError("positions: int64 or int32")
        if positions.shape == (B, T) and not packed:
            pos_b = T
        elif positions.shape != (T,):
            raise ValueError(f"positions: shape ({T},)" + ("" if packed else f" or ({B}, {T})") + f", got {tuple(positions.shape)}")
    elif start < 0 or start + T > table.max_positions:
        raise ValueError(f"positions {start} .. {start + T - 1} leave the table's 0 .. {table.max_positions - 1}")
    d = _device(q, k, positions, table.table)
    _in_use(table, d)
    if out is None:
        yq, yk = q.new_empty(shape), None if k is None else k.new_empty(k.shape)
        lyq, lyk = (yq.data_ptr(), T * H * D, H * D, D), _NONE if k is None else (yk.data_ptr(), T * Hk * D, Hk * D, D)
    else:
        yq, yk = _rotary_out(q, k, out)
        lyq, lyk = _place(yq), _NONE if k is None else _place(yk)
    if B * T == 0:
        return yq, yk
    q = q if q.stride(-1) == 1 else q.contiguous()
    lk = _NONE
    if k is not None:
        k = k if k.stride(-1) == 1 else k.contiguous()
        lk = _place(k)
    at = 0
    if positions is not None:
        if positions.dtype != torch.int64 or not positions.is_contiguous():
            positions = positions.to(torch.int64).contiguous()
        at = positions.data_ptr()
    a = _lib.SEQ_ROTARY_BYTES.pack(*_place(q), *lk, *lyq, *lyk, table.table.data_ptr(), at, pos_b, start, table.max_positions, t, B, T, H, Hk, D,
                                   table.rotary_dim, table.interleaved, transpose)
    _lib.check(_lib.lib().dpc_seq_rotary_run(a, _stream(d)))
    return yq, yk


_NONE = (0, 0, 0, 0)


def _place(x):
    """Address and strides of batch, token, head."""
    s = x.stride()
    return (x.data_ptr(), *s[:3]) if len(s) == 4 else (x.data_ptr(), 0, s[0], s[1])


def _rotary_out(q, k, out):
    """Checks the caller's buffers: an input itself, or something that shares no element with any input or the other buffer."""
    ys = [out] if k is None and torch.is_tensor(out) else list(out)[:1 if k is None else None]
    xs = [q] if k is None else [q, k]
    if len(ys) != len(xs):
        raise ValueError("out: one buffer per tensor")
    for y, x in zip(ys, xs):
        if y.shape != x.shape or y.dtype != x.dtype or y.device != x.device:
            raise ValueError("out: shape, type and device of the input")
        if y.numel() and (y.stride(-1) != 1 or not _distinct(y)):
            raise ValueError("out: the last axis must be contiguous and elements distinct")
        for z in xs:
            itself = z is x and y.data_ptr() == z.data_ptr() and y.stride() == z.stride()
            if not itself and _overlap(y, z):
                raise ValueError("out: a buffer that overlaps an input must be that input")
    if k is not None and _overlap(*ys):
        raise ValueError("out: the two buffers overlap")
    return ys[0], None if k is None else ys[1]


def rotary_forward(q, k, table, positions=None, start=0, out=None):
    """Turns the pairs of every head of q and k (k may be None) by their token's position -> (q', k').

    q, k: [B, T, H, D] / [B, T, Hk, D], or packed [T, H, D] / [T, Hk, D]; the first table.rotary_dim elements of a head are turned, the
    rest is copied.  positions: int64 / int32 [T] or [B, T] on the device, or None: start, start + 1, ...  A position outside the table
    gives NaN in the turned elements (device values cannot be refused without a synchronisation).  out: (q', k') buffers; the inputs
    themselves are allowed."""
    return _rotary(q, k, table, positions, start, out, False)


def rotary_backward(dq, dk, table, positions=None, start=0, out=None):
    """Gradient of `rotary_forward`: the transposed turn of dq and dk (dk may be None)."""
    return _rotary(dq, dk, table, positions, start, out, True)


# ------------------------------------------------------------------------------------------------------------------ attention
class SequencePlan(_Tables):
    """Sequences of different lengths for `attention_forward` / `attention_backward`: checked here, laid out once, used for many calls.

    `packed`: q is [sum(q_lengths), H, D], the sequences one behind the other; k and v alike.  `padded`: q is [B, q_max, H, D], sequence b
    in the first q_lengths[b] rows of its batch entry.  k_lengths default to q_lengths.  Lengths may be zero."""

    def __init__(self, q_lengths, k_lengths, q_max, k_max, device):
        ql = [int(v) for v in q_lengths]
        kl = ql if k_lengths is None else [int(v) for v in k_lengths]
        if len(ql) != len(kl) or not ql:
            raise ValueError("one query length and one key length per sequence, at least one sequence")
        if min(ql) < 0 or min(kl) < 0:
            raise ValueError("lengths must not be negative")
        if sum(ql) >= 2 ** 31 or sum(kl) >= 2 ** 31:
            raise ValueError("too many tokens")
        self.packed_layout = q_max is None
        if not self.packed_layout:
            q_max, k_max = int(q_max), int(q_max if k_max is None else k_max)
            if max(ql) > q_max or max(kl) > k_max:
                raise ValueError("a length exceeds the padded one")
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("libdpc needs device tensors (there is no CPU implementation)")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a SequencePlan copies its tables to the device: build it before the capture")
        self.q_lengths, self.k_lengths, self.q_max, self.k_max = tuple(ql), tuple(kl), q_max, k_max
        self.q_whole = self.packed_layout or min(ql) == q_max          # every row of q belongs to a sequence
        self.k_whole = self.packed_layout or min(kl) == k_max
        rows, q0, k0 = [], 0, 0
        for a, b in zip(ql, kl):
            rows.append((q0, a, k0, b, 0, 0))
            if self.packed_layout:
                q0, k0 = q0 + a, k0 + b
        # block lists: of queries and of keys, for full and for causal scores
        lists = [[e + rows[e[0]] for e in self._tiles(ql, kl, keys, causal)] for causal in (False, True) for keys in (False, True)]
        self.table = torch.tensor([e for t in lists for e in t] or [(0,) * 8], dtype=torch.int32).to(device)
        self._settle()
        self.counts = (len(lists[0]), len(lists[1]))
        q, k = (32 * n for n in self.counts)
        self.offsets = ((0, q), (q + k, q + k + q))                             # of the lists in the table (bytes), by causal
        self.q_longest, self.k_longest, self.q_total, self.k_total = max(ql), max(kl), sum(ql), sum(kl)

    @staticmethod
    def _tiles(ql, kl, keys, causal):
        """(sequence, block of 128) of every block of queries (or keys): in four classes of work, most first, within a class sequence by sequence."""
        blocks = []
        for b, (nq, nk) in enumerate(zip(ql, kl)):
            for t in range(((nk if keys else nq) + 127) // 128):
                if keys:
                    work = nq - max(0, 128 * t - (nk - nq)) if causal else nq
                else:
                    work = min(nk, 128 * (t + 1) + nk - nq) if causal else nk
                blocks.append((max(0, work), b, t))
        most = max((w for w, _, _ in blocks), default=0) or 1
        order = sorted(blocks, key=lambda e: (-(4 * e[0] // (most + 1)), -(kl if not keys else ql)[e[1]], e[1], -e[0]))
        return [(b, t) for _, b, t in order]

    @classmethod
    def packed(cls, q_lengths, k_lengths=None, device="cuda"):
        return cls(q_lengths, k_lengths, None, None, device)

    @classmethod
    def padded(cls, q_lengths, q_max, k_lengths=None, k_max=None, device="cuda"):
        return cls(q_lengths, k_lengths, q_max, k_max, device)


def _attention_args(q, k, v, causal, scale, key_mask, plan):
    """Checks the inputs -> (device; q, k, v in layouts a kernel can read, each with address and strides; the lse's shape; the rest of dpc_seq_attn)."""
    t = _type(q, k, v)
    packed = plan is not None and plan.packed_layout
    if q.dim() != (3 if packed else 4) or k.dim() != q.dim():
        raise ValueError("expected " + ("packed [tokens, heads, head_dim]" if packed else "[batch, tokens, heads, head_dim]") + " tensors")
    if k.shape != v.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must have one shape")
    B, Tq, H, D = (1, *q.shape) if packed else q.shape
    Bk, Tk, Hk, Dk = (1, *k.shape) if packed else k.shape
    if Dk != D or Hk < 1 or H < 1 or H % Hk:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)}: one head size, query heads a multiple of the key heads")
    if D & 7 or not 8 <= D <= 128:
        raise ValueError(f"head size {D}: multiples of 8 up to 128 are supported")
    if B != Bk:
        raise ValueError("q and k must have one batch size")
    if (B | Tq | Tk | H) >> 31:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)}: axes of 2^31 or more are not supported")
    scale = D ** -0.5 if scale is None else float(scale)
    if not 2.0 ** -126 <= scale < 2.0 ** 127:
        raise ValueError("scale must be positive and finite (2^-126 to 2^127)")
    if key_mask is not None and (key_mask.dtype != torch.bool or key_mask.shape != k.shape[:-2]):
        raise ValueError(f"key_mask: bool of shape {tuple(k.shape[:-2])}")
    d = _device(q, k, v, key_mask, plan and plan.table)
    if plan is None:
        blocks, sizes, n_seq, q_len, k_len = (0, 0), (0, 0), B, Tq, Tk
    else:
        n_seq, q_len, k_len = len(plan.q_lengths), plan.q_longest, plan.k_longest
        want = ((1, plan.q_total), (1, plan.k_total)) if packed else ((n_seq, plan.q_max), (n_seq, plan.k_max))
        if ((B, Tq), (Bk, Tk)) != want:
            raise ValueError(f"the plan is for q {want[0]} and k {want[1]} (batch, tokens), got {(B, Tq)} and {(Bk, Tk)}")
        _in_use(plan, d)
        at, (of_q, of_k) = plan.table.data_ptr(), plan.offsets[1 if causal else 0]
        blocks, sizes = (at + of_q, at + of_k), plan.counts
    if key_mask is not None:
        key_mask = key_mask.contiguous()
    es = _BYTES[t]
    lse_b, mask_b = (0, 0) if packed else (H * Tq, Tk)
    tail = (0 if key_mask is None else key_mask.data_ptr(), mask_b, *blocks, *sizes, _TYPE[t], n_seq, H, Hk, D, q_len, k_len, 1 if causal else 0,
            B * H * Tq, scale)
    return d, _lay(q, es), _lay(k, es), _lay(v, es), ((H, Tq) if packed else (B, H, Tq)), (lse_b, Tq), tail, key_mask


_ABSENT = (0,) * 16


def attention_forward(q, k, v, *, causal=False, scale=None, key_mask=None, plan=None, out=None):
    """softmax(scale q k^T) v over the visible keys -> (out, lse).

    q [B, Lq, H, D], k and v [B, Lk, Hk, D] (or packed, see `SequencePlan`), H a multiple of Hk: query head h reads key / value head
    h // (H / Hk); D a multiple of 8 up to 128; scale defaults to D^-0.5.  causal: query i sees keys j <= i + Lk - Lq of its sequence.
    key_mask: bool [B, Lk] (packed: [tokens]), True = takes part; what masked keys and values hold never matters.  A query that sees nothing
    gives zeros and lse -inf.  lse [B, H, Lq] (packed: [H, tokens]) float32 is the log of the softmax's denominator, which
    `attention_backward` needs.  Any strides; layouts whose head rows do not start on 16 bytes are copied first.  Rows of a padded plan that
    belong to no sequence are zero (lse -inf), or left as they were in a given `out` buffer.

    Large values: a NaN or infinity in a key or value that some query of the call sees may reach queries that the causal mask keeps from it, as
    0 * NaN does in the formula.  float32 operands are split into bfloat16 parts: an infinity or a value above 3.38e38 gives NaN.  Scores are
    held in 32 bits: probabilities are off by up to 2^-22 times the score, relative, and scores beyond 2^30 may make their query NaN."""
    if _elsewhere(q):
        with torch.cuda.device(q.device):
            return attention_forward(q, k, v, causal=causal, scale=scale, key_mask=key_mask, plan=plan, out=out)
    d, lq, lk, lv, lse_shape, lse_strides, tail, key_mask = _attention_args(q, k, v, causal, scale, key_mask, plan)
    whole = plan is None or plan.q_whole
    if out is None:
        out = (q.new_empty if whole else q.new_zeros)(q.shape)
    else:
        _device(q, out)
        _written(out, q, "out", (q, k, v))
    lse = q.new_empty(lse_shape, dtype=torch.float32)
    if not whole:
        lse.fill_(-math.inf)
    if lse.numel() == 0:
        return out, lse
    es = _BYTES[q.dtype]
    a = _lib.SEQ_ATTN_BYTES.pack(*lq[1:], *lk[1:], *lv[1:], *_lay(out, es)[1:], lse.data_ptr(), *lse_strides, *_ABSENT, *tail)
    L = _lib.lib()
    nbytes = L.dpc_seq_attn_workspace_bytes(a, 0)
    ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _lib.check(L.dpc_seq_attn_fwd(a, ws.data_ptr() if nbytes else None, nbytes, _stream(d)))
    return out, lse


def attention_backward(dout, q, k, v, out, lse, *, causal=False, scale=None, key_mask=None, plan=None, grads=None):
    """Gradients of `attention_forward` -> (dq, dk, dv); the other arguments as in the forward call, out and lse what it returned.  Rows of a
    padded plan that belong to no sequence get zeros, or stay as they were in given buffers.

    The probabilities are computed again from q, k and lse.  Gradients of a key / value head are summed over the query heads that read it.  Masked
    keys get zero gradients.  grads: buffers for (dq, dk, dv), e.g. views of one packed projection gradient; they must not overlap."""
    if _elsewhere(q):
        with torch.cuda.device(q.device):
            return attention_backward(dout, q, k, v, out, lse, causal=causal, scale=scale, key_mask=key_mask, plan=plan, grads=grads)
    t = _type(q, dout, out)
    if dout.shape != q.shape or out.shape != q.shape:
        raise ValueError(f"dout {tuple(dout.shape)} and out {tuple(out.shape)} must have q's shape {tuple(q.shape)}")
    d, lq, lk, lv, lse_shape, lse_strides, tail, key_mask = _attention_args(q, k, v, causal, scale, key_mask, plan)
    _device(q, dout, out, lse)
    if lse.shape != lse_shape or lse.dtype != torch.float32 or not lse.is_contiguous():
        raise ValueError(f"lse: the contiguous float32 {lse_shape} of attention_forward")
    if grads is None:
        dq = (q.new_empty if plan is None or plan.q_whole else q.new_zeros)(q.shape)
        new = k.new_empty if plan is None or plan.k_whole else k.new_zeros
        dk, dv = new(k.shape), new(k.shape)
    else:
        dq, dk, dv = grads
        _device(q, dq, dk, dv)
        for name, g, like in (("dq", dq, q), ("dk", dk, k), ("dv", dv, v)):
            _written(g, like, name, (q, k, v, dout, out))
        if _overlap(dq, dk) or _overlap(dq, dv) or _overlap(dk, dv):
            raise ValueError("grads: the buffers overlap")
    if lse.numel() == 0 and k.numel() == 0:
        return dq, dk, dv
    es = _BYTES[t]
    lout, ldout = _lay(out, es), _lay(dout, es)
    a = _lib.SEQ_ATTN_BYTES.pack(*lq[1:], *lk[1:], *lv[1:], *lout[1:], lse.data_ptr(), *lse_strides, *ldout[1:], *_lay(dq, es)[1:], *_lay(dk, es)[1:],
                                 *_lay(dv, es)[1:], *tail)
    L = _lib.lib()
    nbytes = L.dpc_seq_attn_workspace_bytes(a, 1)
    ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _lib.check(L.dpc_seq_attn_bwd(a, ws.data_ptr() if nbytes else None, nbytes, _stream(d)))
    return dq, dk, dv
