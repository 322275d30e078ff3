"""The 8-bit inter-step cache: StepCache (src/model/cache.rs:25-81) in e4m3
with a scale for each block of positions and kv head.

  store      K and V rows are quantised as they are written   (ca_kv8_store)
  load       rows are read back as bf16 or fp32               (ca_kv8_load)
  attention  attention over the cache as it is held           (ca_attention_kv8_dev)
  attention_block  norms, RoPE, store and attention of a step (ca_attention_block_kv8_dev)

Each call has a `make_*_args` form for programs that keep their buffers: the
argument block is built once and `*_args(a, stream)` launches it. All calls
are asynchronous on `stream` (None: the legacy default stream) and allocate
nothing, except for scratch that is not passed: `attention` and
`attention_block` make it on the stream that they launch on, `make_*_args` on
torch's current stream, which the first launch on another stream waits for.
Like every tensor of a call, the arguments are to be kept until the work that
was launched with them is done.
"""
from __future__ import annotations

import contextlib
import ctypes
from dataclasses import dataclass
from typing import Any, Optional

from . import CaError, _check, _ptr, _stream, lib

TICKET_BYTES = 4096
BLOCK_TOKENS = (16, 32, 64, 128)


class CaKv8Cache(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scale", ctypes.c_void_p),
                ("v_scale", ctypes.c_void_p), ("batch", ctypes.c_int32),
                ("n_total", ctypes.c_int32), ("n_head_kv", ctypes.c_int32),
                ("head_dim", ctypes.c_int32), ("block_tokens", ctypes.c_int32),
                ("row_stride", ctypes.c_int64)]


class CaKv8StoreArgs(ctypes.Structure):
    _fields_ = [("cache", CaKv8Cache), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p),
                ("n_active", ctypes.c_int32), ("active_pos", ctypes.c_void_p),
                ("cu_active", ctypes.c_void_p), ("total_active", ctypes.c_int64),
                ("kv_len", ctypes.c_void_p), ("status", ctypes.c_void_p)]


class CaKv8LoadArgs(ctypes.Structure):
    _fields_ = [("cache", CaKv8Cache), ("pos", ctypes.c_void_p), ("n_pos", ctypes.c_int32),
                ("k_out", ctypes.c_void_p), ("v_out", ctypes.c_void_p),
                ("out_f32", ctypes.c_int32), ("status", ctypes.c_void_p)]


class CaAttnKv8Args(ctypes.Structure):
    _fields_ = [("cache", CaKv8Cache), ("q", ctypes.c_void_p), ("out", ctypes.c_void_p),
                ("out_f32", ctypes.c_int32), ("q_row_stride", ctypes.c_int64),
                ("out_row_stride", ctypes.c_int64), ("n_head", ctypes.c_int32),
                ("sq", ctypes.c_int32), ("cu_q", ctypes.c_void_p), ("max_sq", ctypes.c_int32),
                ("total_q", ctypes.c_int64), ("q_pos", ctypes.c_void_p),
                ("kv_len", ctypes.c_void_p), ("sliding_window", ctypes.c_int64),
                ("causal_prefix", ctypes.c_int64), ("seq_prefix", ctypes.c_void_p),
                ("scale", ctypes.c_float), ("softcap", ctypes.c_float),
                ("status", ctypes.c_void_p), ("workspace", ctypes.c_void_p),
                ("workspace_bytes", ctypes.c_int64)]


class CaBlockKv8Args(ctypes.Structure):
    _fields_ = [("cache", CaKv8Cache), ("q", ctypes.c_void_p), ("k", ctypes.c_void_p),
                ("v", ctypes.c_void_p), ("n_head", ctypes.c_int32), ("n_active", ctypes.c_int32),
                ("active_pos", ctypes.c_void_p), ("cu_active", ctypes.c_void_p),
                ("max_active", ctypes.c_int32), ("total_active", ctypes.c_int64),
                ("held", ctypes.c_void_p), ("kv_len", ctypes.c_void_p),
                ("q_norm_w", ctypes.c_void_p), ("k_norm_w", ctypes.c_void_p),
                ("v_norm", ctypes.c_int32), ("rms_eps", ctypes.c_float),
                ("rope", ctypes.c_void_p), ("rope_len", ctypes.c_int32),
                ("rope_dim", ctypes.c_int32), ("work", ctypes.c_void_p), ("out", ctypes.c_void_p),
                ("out_f32", ctypes.c_int32), ("out_row_stride", ctypes.c_int64),
                ("sliding_window", ctypes.c_int64), ("causal_prefix", ctypes.c_int64),
                ("seq_prefix", ctypes.c_void_p), ("scale", ctypes.c_float),
                ("softcap", ctypes.c_float), ("status", ctypes.c_void_p),
                ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_int64)]


for _name, _args in (("ca_kv8_store", CaKv8StoreArgs), ("ca_kv8_load", CaKv8LoadArgs),
                     ("ca_attention_kv8_dev", CaAttnKv8Args),
                     ("ca_attention_block_kv8_dev", CaBlockKv8Args)):
    _f = getattr(lib, _name)
    _f.argtypes = [ctypes.POINTER(_args), ctypes.c_void_p]
    _f.restype = ctypes.c_int
lib.ca_attention_kv8_workspace.argtypes = [ctypes.POINTER(CaAttnKv8Args)]
lib.ca_attention_kv8_workspace.restype = ctypes.c_int64


def _torch_stream(stream, device):
    """torch's object for the stream that a launch with `stream` goes to."""
    import torch
    handle = _stream(stream)
    if not handle:
        return torch.cuda.default_stream(device)
    return torch.cuda.ExternalStream(handle, device=device)


def _scratch_on(stream, x, needed):
    """A context in which torch allocates on the stream of a launch, so that
    scratch is cleared before its kernels run there and, once dropped, goes to
    none but later work of that stream."""
    if not needed or not x.is_cuda:
        return contextlib.nullcontext()
    import torch
    return torch.cuda.stream(_torch_stream(stream, x.device))


class _Made:
    """Scratch that a make_*_args call made on torch's current stream: where
    and when, for launches on other streams."""

    def __init__(self, device):
        import torch
        here = torch.cuda.current_stream(device)
        self.device, self.ordered = device, {here.cuda_stream}
        # In a capture the scratch belongs to the graph, as its launches do.
        self.event = None if torch.cuda.is_current_stream_capturing() else here.record_event()

    def before(self, stream):
        """Orders what is launched on `stream` next after the scratch."""
        handle = _stream(stream) or 0
        if handle in self.ordered or self.event is None:
            return
        import torch
        to = _torch_stream(stream, self.device)
        with torch.cuda.stream(to):
            # A capture cannot wait for work outside it; beginning one after
            # the scratch was cleared is the caller's part (torch.cuda.graph
            # waits for the device).
            if torch.cuda.is_current_stream_capturing():
                return
        to.wait_event(self.event)
        self.ordered.add(handle)


def _after_scratch(a, stream):
    made = getattr(a, "_made", None)
    if made is not None:
        made.before(stream)


@dataclass
class Kv8Cache:
    """The cache's tensors: k, v uint8 [batch, n_total, n_head_kv, head_dim]
    (dense but for the stride between positions), k_scale, v_scale fp32
    [batch, ceil(n_total / block_tokens), n_head_kv]."""
    k: Any
    v: Any
    k_scale: Any
    v_scale: Any
    block_tokens: int = 32

    @classmethod
    def alloc(cls, batch: int, n_total: int, n_head_kv: int, head_dim: int, *,
              block_tokens: int = 32, device="cuda") -> "Kv8Cache":
        """An empty cache (zeros: scale 0 means that nothing was written)."""
        import torch
        z = lambda *s, t: torch.zeros(*s, dtype=t, device=device)  # noqa: E731
        n_blocks = -(-n_total // block_tokens)
        return cls(z(batch, n_total, n_head_kv, head_dim, t=torch.uint8),
                   z(batch, n_total, n_head_kv, head_dim, t=torch.uint8),
                   z(batch, n_blocks, n_head_kv, t=torch.float32),
                   z(batch, n_blocks, n_head_kv, t=torch.float32), block_tokens)

    def to_c(self) -> CaKv8Cache:
        b, n, h, d = (int(x) for x in self.k.shape)
        if self.block_tokens not in BLOCK_TOKENS:
            raise ValueError(f"block_tokens must be one of {BLOCK_TOKENS}")
        n_blocks = -(-n // self.block_tokens)
        for name in ("k", "v"):
            x = getattr(self, name)
            if x.element_size() != 1 or tuple(x.shape) != (b, n, h, d):
                raise ValueError(f"{name} must hold bytes of shape {(b, n, h, d)}")
            if x.stride(3) != 1 or x.stride(2) != d or (b > 1 and x.stride(0) != n * x.stride(1)) \
                    or x.stride(1) != self.k.stride(1):
                raise ValueError(f"{name}: only the stride between positions may differ from dense")
        for name in ("k_scale", "v_scale"):
            x = getattr(self, name)
            if str(x.dtype) != "torch.float32" or tuple(x.shape) != (b, n_blocks, h) \
                    or not x.is_contiguous():
                raise ValueError(f"{name} must be contiguous float32 of shape {(b, n_blocks, h)}")
        return CaKv8Cache(_ptr(self.k), _ptr(self.v), _ptr(self.k_scale), _ptr(self.v_scale), b, n,
                          h, d, int(self.block_tokens),
                          int(self.k.stride(1)) if n > 1 or b > 1 else 0)


def _rows(name, x, dtypes, heads, head_dim):
    """[..., heads, head_dim] tensors of whole rows: dtype and layout."""
    if str(x.dtype) not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(dtypes)}")
    if tuple(x.shape[-2:]) != (heads, head_dim) or not x.is_contiguous():
        raise ValueError(f"{name} must be contiguous [..., {heads}, {head_dim}]")
    return x.numel() // (heads * head_dim)


def _i32(name, x, n):
    if x is None:
        return None
    if str(x.dtype) != "torch.int32" or x.numel() != n or not x.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32 with {n} entries")
    return x


def make_store_args(cache: Kv8Cache, k, v, active_pos, *, cu_active=None, kv_len=None,
                    status=None) -> CaKv8StoreArgs:
    """k, v: bf16 [batch, n_active, n_head_kv, head_dim], or [rows, n_head_kv,
    head_dim] with cu_active; active_pos: their positions, ascending within
    each sequence; kv_len: positions each sequence held before."""
    c = cache.to_c()
    rows = _rows("k", k, ("torch.bfloat16",), c.n_head_kv, c.head_dim)
    if _rows("v", v, ("torch.bfloat16",), c.n_head_kv, c.head_dim) != rows:
        raise ValueError("k and v must have the same rows")
    if cu_active is None and c.batch and rows % c.batch:
        raise ValueError("rows must be the same for every sequence (or pass cu_active)")
    _i32("active_pos", active_pos, rows)
    _i32("cu_active", cu_active, c.batch + 1)
    _i32("kv_len", kv_len, c.batch)
    a = CaKv8StoreArgs(c, _ptr(k), _ptr(v), rows // max(c.batch, 1), _ptr(active_pos),
                       _ptr(cu_active), rows if cu_active is not None else 0, _ptr(kv_len),
                       _ptr(status))
    a._keep = (cache, k, v, active_pos, cu_active, kv_len, status)
    return a


def store_args(a: CaKv8StoreArgs, stream=None) -> None:
    _check(lib.ca_kv8_store(ctypes.byref(a), _stream(stream)), "ca_kv8_store")


def store(cache: Kv8Cache, k, v, active_pos, *, stream=None, **kw) -> None:
    """ca_kv8_store: quantise rows into the cache (see make_store_args)."""
    store_args(make_store_args(cache, k, v, active_pos, **kw), stream)


def make_load_args(cache: Kv8Cache, k_out, v_out, pos=None, *, status=None) -> CaKv8LoadArgs:
    """k_out, v_out: bf16 or fp32 [batch, n_pos, n_head_kv, head_dim] (one of
    them may be None); pos: int32 [batch, n_pos], or None for 0 .. n_pos - 1."""
    c = cache.to_c()
    kinds = ("torch.bfloat16", "torch.float32")
    outs = [x for x in (k_out, v_out) if x is not None]
    if not outs:
        raise ValueError("k_out or v_out is needed")
    rows = {_rows("k_out / v_out", x, kinds, c.n_head_kv, c.head_dim) for x in outs}
    if len(rows) != 1 or len({x.dtype for x in outs}) != 1:
        raise ValueError("k_out and v_out must have the same rows and dtype")
    n = rows.pop()
    if c.batch and n % c.batch:
        raise ValueError("rows must be the same for every sequence")
    _i32("pos", pos, n)
    a = CaKv8LoadArgs(c, _ptr(pos), n // max(c.batch, 1), _ptr(k_out), _ptr(v_out),
                      1 if str(outs[0].dtype) == "torch.float32" else 0, _ptr(status))
    a._keep = (cache, k_out, v_out, pos, status)
    return a


def load_args(a: CaKv8LoadArgs, stream=None) -> None:
    _check(lib.ca_kv8_load(ctypes.byref(a), _stream(stream)), "ca_kv8_load")


def load(cache: Kv8Cache, k_out, v_out, pos=None, *, stream=None, **kw) -> None:
    """ca_kv8_load: read rows back (see make_load_args)."""
    load_args(make_load_args(cache, k_out, v_out, pos, **kw), stream)


def workspace_bytes(a: CaAttnKv8Args) -> int:
    """ca_attention_kv8_workspace: bytes that a call with these arguments uses."""
    n = int(lib.ca_attention_kv8_workspace(ctypes.byref(a)))
    if n < 0:
        raise CaError(n, "ca_attention_kv8_workspace")
    return n


def make_attention_args(q, cache: Kv8Cache, out, *, q_pos=None, kv_len=None, cu_q=None, max_sq=0,
                        sliding_window: Optional[int] = None, causal_prefix: Optional[int] = None,
                        seq_prefix=None, scale=1.0, softcap=0.0, status=None,
                        workspace=None) -> CaAttnKv8Args:
    """q: bf16 [batch, sq, n_head, head_dim], or [total_q, n_head, head_dim]
    with cu_q and max_sq; out: the same shape, bf16 or fp32. q and out may
    have any stride between tokens. workspace: device bytes, zeroed once when
    allocated; None: allocated here and kept with the arguments; False: none."""
    c = cache.to_c()
    heads, hd = int(q.shape[-2]), int(q.shape[-1])
    if hd != c.head_dim or str(q.dtype) != "torch.bfloat16":
        raise ValueError("q must be bfloat16 with the cache's head_dim")
    if tuple(out.shape) != tuple(q.shape) or \
            str(out.dtype) not in ("torch.bfloat16", "torch.float32"):
        raise ValueError("out must be bfloat16 or float32 of q's shape")
    want = 3 if cu_q is not None else 4
    if q.dim() != want or (want == 4 and int(q.shape[0]) != c.batch):
        raise ValueError("q must be [batch, sq, n_head, head_dim], or [rows, n_head, head_dim] "
                         "with cu_q")
    strides = []
    for name, x in (("q", q), ("out", out)):
        rs = int(x.stride(-3))
        if x.stride(-1) != 1 or x.stride(-2) != hd or \
                (want == 4 and c.batch > 1 and x.stride(0) != int(x.shape[1]) * rs):
            raise ValueError(f"{name}: only the stride between tokens may differ from dense")
        strides.append(rs if x.shape[-3] > 1 or (want == 4 and c.batch > 1) else 0)
    total = int(q.shape[0]) if want == 3 else int(q.shape[0]) * int(q.shape[1])
    if cu_q is not None and total > c.batch * int(max_sq):
        raise ValueError("max_sq must be the largest query count of a sequence")
    _i32("q_pos", q_pos, total)
    _i32("kv_len", kv_len, c.batch)
    _i32("cu_q", cu_q, c.batch + 1)
    _i32("seq_prefix", seq_prefix, c.batch)
    a = CaAttnKv8Args(c, _ptr(q), _ptr(out), 1 if str(out.dtype) == "torch.float32" else 0,
                      strides[0], strides[1], heads, 0 if want == 3 else int(q.shape[1]),
                      _ptr(cu_q), int(max_sq), total if want == 3 else 0, _ptr(q_pos),
                      _ptr(kv_len), -1 if sliding_window is None else int(sliding_window),
                      -1 if causal_prefix is None else int(causal_prefix), _ptr(seq_prefix),
                      float(scale), float(softcap), _ptr(status), None, 0)
    a._made = None
    if workspace is None:
        n = workspace_bytes(a)
        if n:
            import torch
            workspace = torch.zeros(n, dtype=torch.uint8, device=q.device)
            a._made = _Made(q.device) if q.is_cuda else None
    if workspace is not None and workspace is not False:
        a.workspace, a.workspace_bytes = _ptr(workspace), workspace.numel() * \
            workspace.element_size()
    a._keep = (cache, q, out, q_pos, kv_len, cu_q, seq_prefix, status, workspace)
    return a


def attention_args(a: CaAttnKv8Args, stream=None) -> None:
    _after_scratch(a, stream)
    _check(lib.ca_attention_kv8_dev(ctypes.byref(a), _stream(stream)), "ca_attention_kv8_dev")


def attention(q, cache: Kv8Cache, out, *, stream=None, **kw) -> None:
    """ca_attention_kv8_dev: attention over the cache (see make_attention_args)."""
    with _scratch_on(stream, q, kw.get("workspace") is None):
        a = make_attention_args(q, cache, out, **kw)
    attention_args(a, stream)


def make_block_args(q, k, v, cache: Kv8Cache, out, *, active_pos, rope, rope_len: int,
                    rope_dim: int, work=None, cu_active=None, max_active=0, held=None, kv_len=None,
                    q_norm_w=None, k_norm_w=None, v_norm=False, rms_eps=1e-6,
                    sliding_window: Optional[int] = None, causal_prefix: Optional[int] = None,
                    seq_prefix=None, scale=1.0, softcap=0.0, status=None,
                    workspace=None) -> CaBlockKv8Args:
    """q, k, v: post-projection bf16 [batch, n_active, heads, head_dim], or
    [rows, heads, head_dim] with cu_active and max_active; out: q's shape, bf16
    or fp32. rope: the table of build_rope_cache on the device. work (bf16
    scratch) and workspace: made here and kept with the arguments when None."""
    c = cache.to_c()
    heads = int(q.shape[-2])
    rows = _rows("q", q, ("torch.bfloat16",), heads, c.head_dim)
    for name, x in (("k", k), ("v", v)):
        if _rows(name, x, ("torch.bfloat16",), c.n_head_kv, c.head_dim) != rows:
            raise ValueError(f"{name} must have q's rows")
    if cu_active is None and c.batch and rows % c.batch:
        raise ValueError("rows must be the same for every sequence (or pass cu_active)")
    if cu_active is not None and rows > c.batch * int(max_active):
        raise ValueError("max_active must be the largest row count of a sequence")
    if str(rope.dtype) != "torch.float32" or rope.numel() < rope_len * (rope_dim // 2) * 2:
        raise ValueError("rope must be float32 [rope_len, rope_dim / 2, 2]")
    _i32("active_pos", active_pos, rows)
    _i32("cu_active", cu_active, c.batch + 1)
    _i32("held", held, c.batch)
    need = rows * (heads + 2 * c.n_head_kv) * c.head_dim
    made = work is None
    if made:
        import torch
        work = torch.empty(need, dtype=torch.bfloat16, device=q.device)
    if str(work.dtype) != "torch.bfloat16" or work.numel() < need:
        raise ValueError(f"work must be bfloat16 with at least {need} elements")
    # The attention's own checks and workspace.
    t = make_attention_args(q, cache, out, q_pos=active_pos, kv_len=kv_len, cu_q=cu_active,
                            max_sq=max_active, sliding_window=sliding_window,
                            causal_prefix=causal_prefix, seq_prefix=seq_prefix, scale=scale,
                            softcap=softcap, status=status, workspace=workspace)
    a = CaBlockKv8Args(c, _ptr(q), _ptr(k), _ptr(v), heads, t.sq, _ptr(active_pos),
                       _ptr(cu_active), int(max_active), t.total_q, _ptr(held), _ptr(kv_len),
                       _ptr(q_norm_w), _ptr(k_norm_w), 1 if v_norm else 0, float(rms_eps),
                       _ptr(rope), int(rope_len), int(rope_dim), _ptr(work), _ptr(out), t.out_f32,
                       t.out_row_stride, t.sliding_window, t.causal_prefix, _ptr(seq_prefix),
                       float(scale), float(softcap), _ptr(status), t.workspace, t.workspace_bytes)
    a._keep = (t, k, v, active_pos, cu_active, held, q_norm_w, k_norm_w, rope, work, status)
    a._made = t._made
    if made and a._made is None and q.is_cuda:
        a._made = _Made(q.device)
    return a


def block_args(a: CaBlockKv8Args, stream=None) -> None:
    _after_scratch(a, stream)
    _check(lib.ca_attention_block_kv8_dev(ctypes.byref(a), _stream(stream)),
           "ca_attention_block_kv8_dev")


def attention_block(q, k, v, cache: Kv8Cache, out, *, stream=None, **kw) -> None:
    """ca_attention_block_kv8_dev: one layer's step over the cache (see
    make_block_args)."""
    with _scratch_on(stream, q, kw.get("workspace") is None or kw.get("work") is None):
        a = make_block_args(q, k, v, cache, out, **kw)
    block_args(a, stream)
