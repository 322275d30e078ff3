"""The denoising step after the forward, with the per-candidate reductions on
the GPU: Denoiser::process_logits (src/model/sampler.rs:581-593).

The logits of a step stay in HBM. One ca_candidate_stats launch computes, for
every masked position of the block, the greedy token, entropy, top1 - top2
margin and top-1 probability (collect_candidates :720-749, after
suppress_mask_token / suppress_tokens :90-113); only those four values per
candidate come back to the host, where ranking and commit run as in the
reference (update_credit :597-609, rank_candidates :613-656, commit
:658-671, tokens_to_unmask :115-132 through the C ABI in f32).

At temperature > 0 (pick_token :766-806) the tokens come from ca_sample, in a
second launch over the same logits: temperature, top-k, top-p and min-p, one
random number a candidate. Those numbers come from a numpy Generator, so the
draws are not the reference's own RNG stream; neither is Remasking::Random's
shuffle, which takes the same Generator in place of the reference's StdRng.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass, field
from typing import Optional, Sequence

import numpy as np

from . import CaError, _check, _ptr, _stream, lib
from .layer import one_device

COSINE, LINEAR = 0, 1
ENTROPY_EXIT, LOW_CONFIDENCE, MARGIN, CONFIDENCE, ENTROPY_BOUND, RANDOM = range(6)


class CaCandArgs(ctypes.Structure):
    _fields_ = [("logits", ctypes.c_void_p), ("n_vocab", ctypes.c_int64),
                ("row_stride", ctypes.c_int64), ("rows", ctypes.c_void_p),
                ("n_cand", ctypes.c_int32), ("mask_id", ctypes.c_int32),
                ("suppress", ctypes.c_void_p), ("n_suppress", ctypes.c_int32),
                ("want_entropy", ctypes.c_int32), ("want_prob", ctypes.c_int32),
                ("token", ctypes.c_void_p), ("entropy", ctypes.c_void_p),
                ("margin", ctypes.c_void_p), ("prob", ctypes.c_void_p)]


lib.ca_candidate_stats.argtypes = [ctypes.POINTER(CaCandArgs), ctypes.c_void_p]
lib.ca_candidate_stats.restype = ctypes.c_int
lib.ca_tokens_to_unmask.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int64,
                                    ctypes.c_int32]
lib.ca_tokens_to_unmask.restype = ctypes.c_int64


def tokens_to_unmask(step: int, total_steps: int, masked: int, schedule: int) -> int:
    """tokens_to_unmask (src/model/sampler.rs:115-132), f32 as the reference."""
    n = int(lib.ca_tokens_to_unmask(step, total_steps, masked, schedule))
    if n < 0:
        raise CaError(n, "ca_tokens_to_unmask")
    return n


def candidate_stats(logits, rows, token, entropy=None, margin=None, prob=None, *,
                    n_vocab: int, row_stride: int = 0, mask_id: int = -1, suppress=None,
                    want_entropy: bool = True, want_prob: bool = False, stream=None) -> None:
    """ca_candidate_stats on device tensors (see include/canvas_attn.h)."""
    n_sup = 0 if suppress is None else int(suppress.numel())
    a = CaCandArgs(_ptr(logits), int(n_vocab), int(row_stride), _ptr(rows), int(rows.numel()),
                   int(mask_id), _ptr(suppress) if n_sup else None, n_sup,
                   1 if want_entropy else 0, 1 if want_prob else 0, _ptr(token),
                   _ptr(entropy), _ptr(margin), _ptr(prob))
    rc = lib.ca_candidate_stats(ctypes.byref(a), _stream(stream))
    if rc != 0:
        raise CaError(rc, "ca_candidate_stats")


class CaSampleArgs(ctypes.Structure):
    _fields_ = [("logits", ctypes.c_void_p), ("logits_bf16", ctypes.c_int32),
                ("n_rows", ctypes.c_int64), ("n_vocab", ctypes.c_int64),
                ("row_stride", ctypes.c_int64), ("rows", ctypes.c_void_p),
                ("n_cand", ctypes.c_int32), ("mask_id", ctypes.c_int32),
                ("suppress", ctypes.c_void_p), ("n_suppress", ctypes.c_int32),
                ("u", ctypes.c_void_p), ("temperature", ctypes.c_float),
                ("top_k", ctypes.c_int32), ("top_p", ctypes.c_float), ("min_p", ctypes.c_float),
                ("temperature_row", ctypes.c_void_p), ("top_k_row", ctypes.c_void_p),
                ("top_p_row", ctypes.c_void_p), ("min_p_row", ctypes.c_void_p),
                ("token", ctypes.c_void_p), ("prob", ctypes.c_void_p)]


lib.ca_sample.argtypes = [ctypes.POINTER(CaSampleArgs), ctypes.c_void_p]
lib.ca_sample.restype = ctypes.c_int


def make_sample_args(logits, rows, u, token, prob=None, *, n_vocab: Optional[int] = None,
                     temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mask_id: int = -1,
                     suppress=None) -> CaSampleArgs:
    """logits: fp32 or bf16 [n_rows, >= n_vocab], rows of any stride; rows: int32
    [n_cand] (None: row i); u: fp32 [n_cand] in [0, 1); token: int32 [n_cand]
    out; prob: fp32 [n_cand] out or None. temperature, top_k, top_p and min_p
    are numbers, or tensors with an entry for each candidate (fp32; top_k
    int32). suppress: int32 token ids. Kept for programs that keep their
    buffers; sample_args launches it."""
    kind = {"torch.float32": 0, "torch.bfloat16": 1}.get(str(logits.dtype))
    if kind is None or logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits must be float32 or bfloat16 [rows, vocab]")
    v = int(logits.shape[1]) if n_vocab is None else int(n_vocab)
    if v > logits.shape[1]:
        raise ValueError("n_vocab exceeds the logits' columns")
    n = int(token.numel())

    def check(name, x, dtype, count=None):
        if str(x.dtype) != dtype or not x.is_contiguous() or \
                (count is not None and x.numel() != count):
            raise ValueError(f"{name} must be contiguous {dtype}"
                             + ("" if count is None else f" with {count} entries"))

    check("token", token, "torch.int32")
    check("u", u, "torch.float32", n)
    for name, x, dtype in (("rows", rows, "torch.int32"), ("prob", prob, "torch.float32")):
        if x is not None:
            check(name, x, dtype, n)
    if suppress is not None:
        check("suppress", suppress, "torch.int32")
    scalars, tensors = [], []
    for name, x, dtype in (("temperature", temperature, "torch.float32"),
                           ("top_k", top_k, "torch.int32"), ("top_p", top_p, "torch.float32"),
                           ("min_p", min_p, "torch.float32")):
        each = hasattr(x, "data_ptr")
        if each:
            check(name, x, dtype, n)
        tensors.append(x if each else None)
        scalars.append((int if name == "top_k" else float)(0 if each else x))
    if rows is None and n > logits.shape[0]:
        raise ValueError("more candidates than rows")
    if logits.shape[0] > 1 and logits.stride(0) < v:
        raise ValueError("logits: rows must not overlap")
    kept = (logits, rows, u, token, prob, suppress, *tensors)
    one_device(*kept)
    n_sup = 0 if suppress is None else int(suppress.numel())
    a = CaSampleArgs(_ptr(logits), kind, int(logits.shape[0]), v,
                     int(logits.stride(0)) if logits.shape[0] > 1 else 0, _ptr(rows), n,
                     int(mask_id), _ptr(suppress) if n_sup else None, n_sup, _ptr(u),
                     scalars[0], max(min(scalars[1], 0x7fffffff), -1), scalars[2], scalars[3],
                     _ptr(tensors[0]), _ptr(tensors[1]), _ptr(tensors[2]), _ptr(tensors[3]),
                     _ptr(token), _ptr(prob))
    a._keep = kept
    return a


def sample_args(a: CaSampleArgs, stream=None) -> None:
    _check(lib.ca_sample(ctypes.byref(a), _stream(stream)), "ca_sample")


def sample(logits, rows, u, token, prob=None, *, stream=None, **kw) -> None:
    """ca_sample: a token for each candidate row of device logits (see
    make_sample_args and include/canvas_attn.h)."""
    sample_args(make_sample_args(logits, rows, u, token, prob, **kw), stream)


@dataclass
class Candidate:
    pos: int
    token: int
    entropy: float
    margin: float
    prob: float


@dataclass
class StepParams:
    """The Denoiser parameters this step reads (src/model.rs GenerateParams)."""
    remasking: int = LOW_CONFIDENCE
    schedule: int = COSINE
    entropy_threshold: float = 0.0
    confidence_threshold: float = 0.9
    eb_entropy_bound: float = 0.0
    credit_steps: int = 0
    suppress_ids: Sequence[int] = field(default_factory=list)
    temperature: float = 0.0  # 0: the greedy pick
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0


class DenoiseState:
    """The canvas of one sequence: tokens, which positions are masked, and
    the credit counters (sampler.rs:430-481)."""

    def __init__(self, seq: Sequence[int], is_masked: Sequence[bool], mask_id: int):
        self.seq = np.asarray(seq, dtype=np.int32).copy()
        self.is_masked = np.asarray(is_masked, dtype=bool).copy()
        self.n_masked = int(self.is_masked.sum())
        self.mask_id = int(mask_id)
        self.prev_pick = np.full(len(self.seq), -1, dtype=np.int64)
        self.credit = np.zeros(len(self.seq), dtype=np.int64)


def collect_candidates(state: DenoiseState, logits, n_vocab: int, rng: range, shift: int,
                       params: StepParams, stream=None,
                       draw_rng: Optional[np.random.Generator] = None):
    """collect_candidates (sampler.rs:720-749) with the row reductions on the
    GPU. `logits`: device fp32 [len(seq), n_vocab]; its suppressed entries of
    the candidate rows are set to -inf, as process_logits does. At
    params.temperature > 0 token and prob are those of the draw, entropy and
    margin the row's; draw_rng gives the random numbers. Everything runs on
    `stream` (None: the legacy default stream), the copies to the host too."""
    import torch
    pos = [p for p in rng if state.is_masked[p]]
    if not pos:
        return []
    dev = logits.device
    if dev.type == "cuda":
        handle = _stream(stream)
        on = (torch.cuda.ExternalStream(handle, device=dev) if handle
              else torch.cuda.default_stream(dev))
        with torch.cuda.stream(on):
            return _collect(state, logits, n_vocab, pos, shift, params, handle, draw_rng)
    return _collect(state, logits, n_vocab, pos, shift, params, stream, draw_rng)


def _collect(state, logits, n_vocab, pos, shift, params, stream, draw_rng):
    import torch
    dev = logits.device
    rows = torch.tensor([max(p - shift, 0) for p in pos], dtype=torch.int32, device=dev)
    n = len(pos)
    tok = torch.empty(n, dtype=torch.int32, device=dev)
    vals = torch.empty((3, n), dtype=torch.float32, device=dev)
    sup = (torch.tensor(list(params.suppress_ids), dtype=torch.int32, device=dev)
           if len(params.suppress_ids) else None)
    needs_entropy = params.remasking in (ENTROPY_EXIT, LOW_CONFIDENCE, ENTROPY_BOUND)
    needs_prob = params.remasking == CONFIDENCE
    candidate_stats(logits, rows, tok, vals[0], vals[1], vals[2], n_vocab=n_vocab,
                    mask_id=state.mask_id, suppress=sup, want_entropy=needs_entropy,
                    want_prob=needs_prob, stream=stream)
    if params.temperature > 0:
        g = draw_rng or np.random.default_rng()
        u = torch.from_numpy(g.random(n, dtype=np.float32)).to(dev)
        sample(logits, rows, u, tok, vals[2], n_vocab=n_vocab, temperature=params.temperature,
               top_k=params.top_k, top_p=params.top_p, min_p=params.min_p, mask_id=state.mask_id,
               suppress=sup, stream=stream)
    tok_h = tok.cpu().numpy()
    ent, mar, prob = vals.cpu().numpy()
    return [Candidate(p, int(tok_h[i]), float(ent[i]), float(mar[i]), float(prob[i]))
            for i, p in enumerate(pos)]


def update_credit(state: DenoiseState, cands, params: StepParams) -> None:
    """update_credit (sampler.rs:597-609)."""
    if params.credit_steps == 0:
        return
    for c in cands:
        if c.token == state.prev_pick[c.pos]:
            state.credit[c.pos] += 1
        else:
            state.credit[c.pos] = 0
            state.prev_pick[c.pos] = c.token


def rank_candidates(cands, params: StepParams, local_step: int, block_steps: int,
                    rng: Optional[np.random.Generator] = None) -> int:
    """rank_candidates (sampler.rs:613-656): orders `cands` in place (stable
    sorts, as Rust's sort_by) and returns how many to unmask."""
    n = len(cands)
    schedule_n = tokens_to_unmask(local_step, block_steps, n, params.schedule)
    r = params.remasking
    f32 = lambda x: float(np.float32(x))  # noqa: E731  (thresholds are f32 in the reference)
    if r == ENTROPY_EXIT:
        cands.sort(key=lambda c: _total_key(c.entropy))
        easy = _take_while(cands, lambda c: c.entropy < f32(params.entropy_threshold))
        return min(max(schedule_n, easy), n)
    if r == LOW_CONFIDENCE:
        cands.sort(key=lambda c: _total_key(c.entropy))
        return schedule_n
    if r == MARGIN:
        cands.sort(key=lambda c: -_total_key(c.margin))
        return schedule_n
    if r == CONFIDENCE:
        cands.sort(key=lambda c: -_total_key(c.prob))
        confident = _take_while(cands, lambda c: c.prob >= f32(params.confidence_threshold))
        return min(max(schedule_n, confident), n)
    if r == ENTROPY_BOUND:
        cands.sort(key=lambda c: _total_key(c.entropy))
        confident = _take_while(cands, lambda c: c.entropy < f32(params.eb_entropy_bound))
        return min(max(confident, 1), n)
    if r == RANDOM:
        g = rng or np.random.default_rng()
        for i in range(n - 1, 0, -1):
            j = int(g.integers(0, i + 1))
            cands[i], cands[j] = cands[j], cands[i]
        return schedule_n
    raise ValueError(f"unknown remasking {r}")


def _total_key(x: float) -> int:
    """Sort key with the order of Rust's f32::total_cmp (-0.0 < +0.0, NaNs at
    the ends by sign) on the f32 value."""
    b = int(np.array(x, dtype=np.float32).view(np.int32))
    return b ^ ((b >> 31) & 0x7FFFFFFF)


def _take_while(cands, pred) -> int:
    k = 0
    for c in cands:
        if not pred(c):
            break
        k += 1
    return k


def commit(state: DenoiseState, cands, n_unmask: int, params: StepParams) -> int:
    """commit (sampler.rs:658-671): the first n_unmask ranked candidates plus
    any credit-stable ones; returns how many were committed."""
    committed = 0
    for rank, c in enumerate(cands):
        credit_ok = params.credit_steps > 0 and state.credit[c.pos] >= params.credit_steps
        if rank < n_unmask or credit_ok:
            state.seq[c.pos] = c.token
            state.is_masked[c.pos] = False
            state.n_masked -= 1
            committed += 1
    return committed


def process_logits(state: DenoiseState, logits, n_vocab: int, rng: range, shift: int,
                   local_step: int, block_steps: int, params: StepParams,
                   stream=None, shuffle_rng=None) -> int:
    """process_logits (sampler.rs:581-593) after the forward: suppress,
    collect, credit, rank, commit. Returns the number of committed tokens.
    shuffle_rng: the random numbers of Remasking::Random and of the draws at
    params.temperature > 0."""
    cands = collect_candidates(state, logits, n_vocab, rng, shift, params, stream, shuffle_rng)
    update_credit(state, cands, params)
    n_unmask = rank_candidates(cands, params, local_step, block_steps, shuffle_rng)
    return commit(state, cands, n_unmask, params)
