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
captured into graphs.  Nothing is accumulated with atomics: results repeat bit for bit.  Arguments are checked on the host (ValueError /
TypeError / RuntimeError); tensors must live on the GPU (no CPU path)."""
import ctypes as C
import math

import torch

from . import _lib

_TYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


# ------------------------------------------------------------------------------------------------------------------ checks
def _type(*tensors):
    t = tensors[0].dtype
    if t not in _TYPE:
        raise TypeError(f"element type {t}: float32, float16 and bfloat16 are supported")
    for x in tensors[1:]:
        if x.dtype != t:
            raise TypeError(f"one element type per call, got {t} and {x.dtype}")
    return t


def _device(*tensors):
    d = tensors[0].device
    for x in tensors:
        if not x.is_cuda:
            raise RuntimeError("libdpc needs device tensors (there is no CPU implementation)")
        if x.device != d:
            raise RuntimeError(f"tensors on {d} and {x.device}")
    return d


def _stream(device):
    return C.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _in_use(owner):
    """The owner's table is read on the current stream: its memory is not handed on before that stream is done with it."""
    current = torch.cuda.current_stream(owner.table.device)
    if current != owner.stream:
        owner.table.record_stream(current)


def _p(t):
    return C.c_void_p(t.data_ptr()) if t is not None else None


def _rows16(x):
    """x with a contiguous last axis, every other stride and the base on 16 bytes and tokens less than 2^25 bytes apart: itself or a contiguous copy."""
    es = x.element_size()
    if x.numel() == 0:
        return x
    if x.stride(-1) == 1 and x.data_ptr() % 16 == 0 and all(s * es % 16 == 0 for s, n in zip(x.stride()[:-1], x.shape[:-1]) if n > 1):
        if x.shape[-3] == 1 or x.stride(-3) * es < 1 << 25:
            return x
    return x.clone(memory_format=torch.contiguous_format)


def _shares(a, b):
    return a.untyped_storage().data_ptr() == b.untyped_storage().data_ptr()


def _overlap(a, b):
    """Whether a and b may share an element: equal strides and a shift inside one row of the larger axes keep views of one projection apart."""
    if not (a.numel() and b.numel()) or not _shares(a, b):
        return False
    if a.dim() == b.dim() and a.dim() >= 2 and a.stride()[:-2] == b.stride()[:-2]:
        wide = lambda t: (t.shape[-2] - 1) * t.stride(-2) + (t.shape[-1] - 1) * t.stride(-1) + 1
        (lo, wl), (hi, wh) = sorted(((a.storage_offset(), wide(a)), (b.storage_offset(), wide(b))))
        outer = min((s for s, n in zip(a.stride()[:-2], a.shape[:-2]) if n > 1), default=None)
        if hi - lo >= wl and (outer is None or (hi - lo) + wh <= outer):
            return False
    last = lambda t: t.storage_offset() + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return a.storage_offset() <= last(b) and b.storage_offset() <= last(a)


def _written(x, like, name, inputs):
    """Checks a caller's output buffer: shape, type, layout of distinct elements, and no element shared with an input."""
    if x.shape != like.shape or x.dtype != like.dtype:
        raise ValueError(f"{name}: expected shape {tuple(like.shape)} of {like.dtype}, got {tuple(x.shape)} of {x.dtype}")
    order = sorted((s, n) for s, n in zip(x.stride(), x.shape) if n > 1)
    reach = 0
    for s, n in order:
        if s <= reach:
            raise ValueError(f"{name}: elements of the buffer overlap")
        reach += s * (n - 1)
    if x.numel() and _rows16(x) is not x:
        raise ValueError(f"{name}: the last axis must be contiguous, base and strides multiples of 16 bytes")
    if any(_overlap(x, i) for i in inputs):
        raise ValueError(f"{name}: the buffer overlaps an input")


# ------------------------------------------------------------------------------------------------------------------ layer norm
def _norm_params(x, weight, bias):
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.shape != x.shape[-1:]:
            raise ValueError(f"{name}: expected shape {tuple(x.shape[-1:])}, got {tuple(p.shape)}")
        if p.dtype not in (torch.float32, x.dtype):
            raise TypeError(f"{name}: float32 or {x.dtype}, got {p.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("weight and bias must have one type")
    p = weight if weight is not None else bias
    return _TYPE[torch.float32] if p is None else _TYPE[p.dtype]


def _matrix(x):
    """x as [rows, C] with one row stride (a view where the layout allows it, else a copy); broadcast rows are copied."""
    n = x.shape[-1]
    if x.dim() == 2 and x.stride(1) == 1 and (x.shape[0] == 1 or x.stride(0) >= n):
        return x
    y = x.reshape(-1, n)
    if y.stride(1) != 1 or (y.shape[0] > 1 and y.stride(0) < n):
        y = y.clone(memory_format=torch.contiguous_format)
    return y


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5):
    """y = (x - mean) / sqrt(variance + eps) * weight + bias over the last axis (biased variance) -> (y, stats).

    x: any shape [..., C], C >= 1, any strides; weight, bias: [C] of float32 or of x's type, or None.  stats [rows, 2] float32 = (mean,
    1 / sqrt(variance + eps)) is what `layer_norm_backward` needs."""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x: at least one axis of at least one element")
    eps = float(eps)
    if not (eps > 0 and math.isfinite(eps)):
        raise ValueError("eps must be positive and finite")
    t = _TYPE[_type(x)]
    wt = _norm_params(x, weight, bias)
    dev = _device(*[v for v in (x, weight, bias) if v is not None])
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    rows = x.numel() // x.shape[-1]
    stats = torch.empty(rows, 2, dtype=torch.float32, device=dev)
    if rows == 0:
        return y, stats
    with torch.cuda.device(dev):
        m = _matrix(x)
        w, b = (v.contiguous() if v is not None else None for v in (weight, bias))
        _lib.check(_lib.lib().dpc_seq_norm_fwd(_p(m), _p(w), _p(b), _p(y), _p(stats), rows, x.shape[-1], m.stride(0) if rows > 1 else x.shape[-1],
                                               eps, t, wt, _stream(dev)))
    return y, stats


def layer_norm_backward(dy, x, stats, weight=None, param_grads=True, param_dtype=None):
    """Gradients of `layer_norm_forward` -> (dx, dweight, dbias): dx in x's shape, dweight and dbias [C] in weight's type (without a weight:
    `param_dtype`, float32 by default).  param_grads=False skips the two sums (None, None)."""
    if dy.shape != x.shape:
        raise ValueError(f"dy {tuple(dy.shape)} must have x's shape {tuple(x.shape)}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x: at least one axis of at least one element")
    t = _TYPE[_type(x, dy)]
    wt = _norm_params(x, weight, None)
    n = x.shape[-1]
    rows = x.numel() // n
    if stats.shape != (rows, 2) or stats.dtype != torch.float32 or not stats.is_contiguous():
        raise ValueError(f"stats: the contiguous float32 [{rows}, 2] of layer_norm_forward, got {tuple(stats.shape)} of {stats.dtype}")
    pt = weight.dtype if weight is not None else param_dtype or torch.float32
    if pt not in (torch.float32, x.dtype) or (weight is not None and param_dtype not in (None, pt)):
        raise TypeError(f"param_dtype: float32 or {x.dtype}; with a weight, the weight's type")
    if weight is None:
        wt = _TYPE[pt]
    dev = _device(*[v for v in (x, dy, stats, weight) if v is not None])
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
    dw, db = (torch.empty(n, dtype=pt, device=dev) for _ in range(2)) if param_grads else (None, None)
    if rows == 0:
        return dx, dw.zero_() if dw is not None else None, db.zero_() if db is not None else None
    L = _lib.lib()
    with torch.cuda.device(dev):
        mx, mdy = _matrix(x), _matrix(dy)
        w = weight.contiguous() if weight is not None else None
        ws = _lib.workspace(L.dpc_seq_norm_bwd_workspace_bytes(rows, n), dev) if param_grads else None
        _lib.check(L.dpc_seq_norm_bwd(_p(mdy), _p(mx), _p(stats), _p(w), _p(dx), _p(dw), _p(db), rows, n, mdy.stride(0) if rows > 1 else n,
                                      mx.stride(0) if rows > 1 else n, t, wt, _p(ws), ws.numel() if ws is not None else 0, _stream(dev)))
    return dx, dw, db


# ------------------------------------------------------------------------------------------------------------------ rotary positions
class RotaryTable:
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
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("libdpc needs device tensors (there is no CPU implementation)")
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
        self.stream = torch.cuda.current_stream(self.table.device)
        self.stream.synchronize()                                                      # whole for whatever stream uses it


def _as_btd(x):
    """(strides of batch, token, head; batch, tokens) of [B, T, H, D] or packed [T, H, D]."""
    if x.dim() == 4:
        return x.stride()[:3], x.shape[0], x.shape[1]
    return (0,) + x.stride()[:2], 1, x.shape[0]


def _seq_tensor(x):
    if x is None:
        return _lib.SeqTensor(None, 0, 0, 0)
    (b, t, h), _, _ = _as_btd(x)
    n = x.shape if x.dim() == 4 else (1,) + tuple(x.shape)
    return _lib.SeqTensor(x.data_ptr(), *(s if m > 1 else 0 for s, m in zip((b, t, h), n)))


def _rotary(q, k, table, positions, start, out, transpose):
    both = [q] if k is None else [q, k]
    for x in both:
        if x.dim() not in (3, 4):
            raise ValueError("expected [batch, tokens, heads, head_dim] or packed [tokens, heads, head_dim]")
    if k is not None and (k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1]):
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} must agree but for the heads")
    t = _TYPE[_type(*both)]
    D = q.shape[-1]
    if table.rotary_dim > D:
        raise ValueError(f"the table's rotary_dim {table.rotary_dim} exceeds the head's {D}")
    _, B, T = _as_btd(q)
    start = int(start)
    pos_b = 0
    if positions is not None:
        if start != 0:
            raise ValueError("give positions or start, not both")
        if positions.dtype not in (torch.int64, torch.int32):
            raise TypeError("positions: int64 or int32")
        if tuple(positions.shape) not in ((T,), (B, T) if q.dim() == 4 else (T,)):
            raise ValueError(f"positions: shape ({T},)" + (f" or ({B}, {T})" if q.dim() == 4 else "") + f", got {tuple(positions.shape)}")
        if positions.dim() == 2:
            pos_b = T
    elif start < 0 or start + T > table.max_positions:
        raise ValueError(f"positions {start} .. {start + T - 1} leave the table's 0 .. {table.max_positions - 1}")
    dev = _device(table.table, *both, *([positions] if positions is not None else []))
    _in_use(table)
    with torch.cuda.device(dev):
        if out is None:
            ys = [torch.empty(x.shape, dtype=x.dtype, device=dev) for x in both]
        else:
            ys = [out] if k is None and torch.is_tensor(out) else list(out)
            ys = ys[:1] if k is None else ys
            if len(ys) != len(both):
                raise ValueError("out: one buffer per tensor")
            for y, x in zip(ys, both):
                if y.shape != x.shape or y.dtype != x.dtype or y.device != x.device:
                    raise ValueError("out: shape, type and device of the input")
                if y.numel() and y.stride(-1) != 1 or any(s == 0 and n > 1 for s, n in zip(y.stride(), y.shape)):
                    raise ValueError("out: the last axis must be contiguous and elements distinct")
                for z in both:
                    itself = z is x and y.data_ptr() == z.data_ptr() and y.stride() == z.stride()
                    if _shares(y, z) and not itself and _overlap(y, z):
                        raise ValueError("out: a buffer that overlaps an input must be that input")
            if k is not None and _overlap(*ys):
                raise ValueError("out: the two buffers overlap")
        if q.numel() == 0 and (k is None or k.numel() == 0):
            return (ys[0], ys[1] if k is not None else None)
        xs = [x if x.stride(-1) == 1 else x.contiguous() for x in both]
        pos = None if positions is None else positions.to(torch.int64).contiguous()
        a = _lib.SeqRotary(xq=_seq_tensor(xs[0]), yq=_seq_tensor(ys[0]), xk=_seq_tensor(xs[1] if k is not None else None),
                           yk=_seq_tensor(ys[1] if k is not None else None), table=table.table.data_ptr(),
                           positions=pos.data_ptr() if pos is not None else None, pos_stride_b=pos_b, start=start,
                           max_positions=table.max_positions, type=t, batch=B, tokens=T, heads=q.shape[-2], kv_heads=k.shape[-2] if k is not None else 0,
                           head_dim=D, rotary_dim=table.rotary_dim, interleaved=1 if table.layout == "interleaved" else 0, transpose=1 if transpose else 0)
        _lib.check(_lib.lib().dpc_seq_rotary_run(C.byref(a), _stream(dev)))
    return (ys[0], ys[1] if k is not None else None)


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
class SequencePlan:
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
            rows.append((q0, a, k0, b))
            if self.packed_layout:
                q0, k0 = q0 + a, k0 + b
        tiles = [self._tiles(ql, kl), self._tiles(kl, ql)]
        flat = torch.tensor([v for r in rows for v in r] + [v for t in tiles for e in t for v in e], dtype=torch.int32)
        self.table = flat.to(device)                                    # (a blocking copy: whole for whatever stream uses it)
        self.stream = torch.cuda.current_stream(self.table.device)
        self.counts = tuple(len(t) for t in tiles)
        self._offsets = (0, 4 * len(rows), 4 * len(rows) + 2 * len(tiles[0]))

    @staticmethod
    def _tiles(lengths, other):
        """(sequence, block of 128) of every block, those of the longest sequences first."""
        order = sorted(range(len(lengths)), key=lambda b: -min(lengths[b], 1) * other[b])
        return [(b, t) for b in order for t in reversed(range((lengths[b] + 127) // 128))]

    @classmethod
    def packed(cls, q_lengths, k_lengths=None, device="cuda"):
        return cls(q_lengths, k_lengths, None, None, device)

    @classmethod
    def padded(cls, q_lengths, q_max, k_lengths=None, k_max=None, device="cuda"):
        return cls(q_lengths, k_lengths, q_max, k_max, device)

    def _pointer(self, i):
        return self.table.data_ptr() + 4 * self._offsets[i]


def _attention_args(q, k, v, causal, scale, key_mask, plan):
    """Checks the inputs -> (16-byte-row forms of q, k, v; filled dpc_seq_attn; the shape of lse; device)."""
    t = _type(q, k, v)
    packed = plan is not None and plan.packed_layout
    want = 3 if packed else 4
    if q.dim() != want or k.dim() != want or v.dim() != want:
        raise ValueError("expected " + ("packed [tokens, heads, head_dim]" if packed else "[batch, tokens, heads, head_dim]") + " tensors")
    if k.shape != v.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must have one shape")
    H, Hk, D = q.shape[-2], k.shape[-2], q.shape[-1]
    if k.shape[-1] != D or Hk < 1 or H < 1 or H % Hk:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)}: one head size, query heads a multiple of the key heads")
    if D % 8 or not 8 <= D <= 128:
        raise ValueError(f"head size {D}: multiples of 8 up to 128 are supported")
    if not packed and q.shape[0] != k.shape[0]:
        raise ValueError("q and k must have one batch size")
    scale = D ** -0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError("scale must be positive and finite")
    if key_mask is not None:
        if key_mask.dtype != torch.bool or key_mask.shape != k.shape[:-2]:
            raise ValueError(f"key_mask: bool of shape {tuple(k.shape[:-2])}")
    if plan is None:
        B, q_len, k_len = q.shape[0], q.shape[1], k.shape[1]
    else:
        B, q_len, k_len = len(plan.q_lengths), max(plan.q_lengths), max(plan.k_lengths)
        shape = ((sum(plan.q_lengths),), (sum(plan.k_lengths),)) if packed else ((B, plan.q_max), (B, plan.k_max))
        if (tuple(q.shape[:-2]), tuple(k.shape[:-2])) != shape:
            raise ValueError(f"the plan is for q {shape[0]} and k {shape[1]} tokens, got {tuple(q.shape[:-2])} and {tuple(k.shape[:-2])}")
    dev = _device(q, k, v, *([key_mask] if key_mask is not None else []), *([plan.table] if plan is not None else []))
    if plan is not None:
        _in_use(plan)
    if key_mask is not None:
        key_mask = key_mask.contiguous()
    lse_shape = (H, q.shape[0]) if packed else (q.shape[0], H, q.shape[1])
    a = _lib.SeqAttn(key_mask=key_mask.data_ptr() if key_mask is not None else None, mask_stride_b=0 if packed else k.shape[1], type=_TYPE[t], batch=B, heads=H,
                     kv_heads=Hk, head_dim=D, q_len=q_len, k_len=k_len, causal=1 if causal else 0, lse_rows=math.prod(lse_shape), scale=scale,
                     lse_stride_b=0 if packed else H * q.shape[1], lse_stride_h=lse_shape[-1], k_rows=k.numel() // D,
                     k_row_stride_b=0 if packed else Hk * k.shape[1], k_row_stride_h=k.shape[-3])
    if plan is not None:
        a.seqs, a.q_tiles, a.k_tiles = (plan._pointer(i) for i in range(3))
        a.n_q_tiles, a.n_k_tiles = plan.counts
    q, k, v = _rows16(q), _rows16(k), _rows16(v)
    a.q, a.k, a.v = _seq_tensor(q), _seq_tensor(k), _seq_tensor(v)
    return (q, k, v, key_mask), a, lse_shape, dev


def attention_forward(q, k, v, *, causal=False, scale=None, key_mask=None, plan=None, out=None):
    """softmax(scale q k^T) v over the visible keys -> (out, lse).

    q [B, Lq, H, D], k and v [B, Lk, Hk, D] (or packed, see `SequencePlan`), H a multiple of Hk: query head h reads key / value head
    h // (H / Hk); D a multiple of 8 up to 128; scale defaults to D^-0.5.  causal: query i sees keys j <= i + Lk - Lq of its sequence.
    key_mask: bool [B, Lk] (packed: [tokens]), True = takes part; what masked keys and values hold never matters.  A query that sees
    nothing gives zeros and lse -inf.  lse [B, H, Lq] (packed: [H, tokens]) float32 is the log of the softmax's denominator, which
    `attention_backward` needs.  Any strides; layouts whose head rows do not start on 16 bytes are copied first.  Rows of a padded plan
    that belong to no sequence are zero (lse -inf), or left as they were in a given `out` buffer."""
    (q, k, v, key_mask), a, lse_shape, dev = _attention_args(q, k, v, causal, scale, key_mask, plan)
    whole = plan is None or plan.q_whole
    with torch.cuda.device(dev):
        if out is None:
            out = (torch.empty if whole else torch.zeros)(q.shape, dtype=q.dtype, device=dev)
        else:
            _device(q, out)
            _written(out, q, "out", (q, k, v))
        lse = torch.empty(lse_shape, dtype=torch.float32, device=dev)
        if not whole:
            lse.fill_(-math.inf)
        if q.numel() == 0:
            return out, lse
        a.out, a.lse = _seq_tensor(out), lse.data_ptr()
        L = _lib.lib()
        nbytes = L.dpc_seq_attn_workspace_bytes(C.byref(a), 0)
        ws = _lib.workspace(nbytes, dev) if nbytes else None
        _lib.check(L.dpc_seq_attn_fwd(C.byref(a), _p(ws), nbytes, _stream(dev)))
    return out, lse


def attention_backward(dout, q, k, v, out, lse, *, causal=False, scale=None, key_mask=None, plan=None, grads=None):
    """Gradients of `attention_forward` -> (dq, dk, dv); the other arguments as in the forward call, out and lse what it returned.

    The probabilities are computed again from q, k and lse.  Gradients of a key / value head are summed over the query heads that read it.  Masked
    keys get zero gradients.  grads: buffers for (dq, dk, dv), e.g. views of one packed projection gradient; they must not overlap."""
    _type(q, dout, out)
    if dout.shape != q.shape or out.shape != q.shape:
        raise ValueError(f"dout {tuple(dout.shape)} and out {tuple(out.shape)} must have q's shape {tuple(q.shape)}")
    (q, k, v, key_mask), a, lse_shape, dev = _attention_args(q, k, v, causal, scale, key_mask, plan)
    _device(q, dout, out, lse)
    if tuple(lse.shape) != tuple(lse_shape) or lse.dtype != torch.float32 or not lse.is_contiguous():
        raise ValueError(f"lse: the contiguous float32 {tuple(lse_shape)} of attention_forward")
    with torch.cuda.device(dev):
        dout, out = _rows16(dout), _rows16(out)
        if grads is None:
            dq = (torch.empty if plan is None or plan.q_whole else torch.zeros)(q.shape, dtype=q.dtype, device=dev)
            dk, dv = ((torch.empty if plan is None or plan.k_whole else torch.zeros)(k.shape, dtype=k.dtype, device=dev) for _ in range(2))
        else:
            dq, dk, dv = grads
            _device(q, dq, dk, dv)
            for name, g, like in (("dq", dq, q), ("dk", dk, k), ("dv", dv, v)):
                _written(g, like, name, (q, k, v, dout, out))
            if _overlap(dq, dk) or _overlap(dq, dv) or _overlap(dk, dv):
                raise ValueError("grads: the buffers overlap")
        if q.numel() == 0 and k.numel() == 0:
            return dq, dk, dv
        a.dout, a.out, a.dq, a.dk, a.dv = (_seq_tensor(x) for x in (dout, out, dq, dk, dv))
        a.lse = lse.data_ptr()
        L = _lib.lib()
        nbytes = L.dpc_seq_attn_workspace_bytes(C.byref(a), 1)
        ws = _lib.workspace(nbytes, dev) if nbytes else None
        _lib.check(L.dpc_seq_attn_bwd(C.byref(a), _p(ws), nbytes, _stream(dev)))
    return dq, dk, dv
