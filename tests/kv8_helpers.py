"""Plain restatements of the 8-bit cache's operators for its tests, in 64
bits and straight from their definitions: store_ref walks the blocks one by
one, attention_ref the (sequence, head) pairs."""
from __future__ import annotations

import math

import torch

F8 = torch.float8_e4m3fn


def e4m3_round(x: torch.Tensor) -> torch.Tensor:
    """fp64 to the nearest e4m3 value (ties to even, saturating)."""
    _, e = torch.frexp(x)
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64),
                     (e.double() - 1).clamp(min=-6) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def held_values(held: torch.Tensor, scale: torch.Tensor, T: int) -> torch.Tensor:
    """What uint8 [b, n, h, d] with scales [b, blocks, h] stands for (fp64)."""
    at = torch.arange(held.shape[1], device=held.device) // T
    return held.view(F8).double() * scale.double()[:, at].unsqueeze(-1)


def need_exp(amax: float) -> int:
    if amax == 0:
        return -64
    k = -64
    while amax > 448 * 2.0 ** k and k < 120:
        k += 1
    return k


def store_ref(held, scale, T, new, rows, pos, n_total, held_len):
    """One of K and V, in place: held fp64 e4m3 values [b, n, h, d], scale
    fp64 [b, blocks, h], new fp64 [rows, h, d]; rows: per sequence the range
    of its rows; held_len: per sequence what it held."""
    for b, (r0, r1) in enumerate(rows):
        by_block = {}
        for r in range(r0, r1):
            by_block.setdefault(int(pos[r]) // T, []).append(r)
        for blk, members in by_block.items():
            active = {int(pos[r]) for r in members}
            inside = range(blk * T, min((blk + 1) * T, n_total))
            stays = any(p < held_len[b] and p not in active for p in inside)
            for h in range(held.shape[2]):
                x = new[members, h]
                fin = x[torch.isfinite(x)].abs()
                amax = float(fin.max()) if fin.numel() else 0.0
                need = 2.0 ** need_exp(amax)
                was = float(scale[b, blk, h])
                keep = stays and was > 0
                now = max(was, need) if keep else need
                if keep and now > was:
                    for p in inside:
                        if p not in active:
                            held[b, p, h] = e4m3_round(held[b, p, h] * (was / now))
                scale[b, blk, h] = now
                for r in members:
                    held[b, int(pos[r]), h] = e4m3_round(new[r, h] / now)


def random_cache(g, b, n, h, d, T, device="cpu", spread=2):
    """uint8 values and power-of-two scales as the store leaves them."""
    x = torch.randn(b, n, h, d, generator=g)
    blocks = -(-n // T)
    up = torch.pow(2.0, torch.randint(-spread, spread + 1, (b, blocks, h), generator=g).float())
    at = torch.arange(n) // T
    x = x * up[:, at].unsqueeze(-1)
    pad = torch.zeros(b, blocks * T, h, d)
    pad[:, :n] = x
    amax = pad.view(b, blocks, T, h, d).abs().amax(dim=(2, 4))
    scale = torch.tensor([2.0 ** need_exp(float(a)) for a in amax.flatten()]).view_as(amax)
    held = (x / scale[:, at].unsqueeze(-1)).to(F8).view(torch.uint8)
    return held.to(device), scale.float().to(device)


def attention_ref(q, k, v, pos, length, *, scale, window=None, prefix=None, cap=0.0):
    """One sequence in fp64: q [sq, H, d], k and v [n, Hkv, d] values. Returns
    the output and sum_i p_i |v_i| (what the tolerances are taken against)."""
    sq, H, d = q.shape
    n, hkv = k.shape[:2]
    out = torch.empty(sq, H, d, dtype=torch.float64, device=q.device)
    mag = torch.empty_like(out)
    key = torch.arange(n, device=q.device)
    qp = pos.long().view(-1, 1).to(q.device)
    see = (key < length).expand(sq, n)
    if window is not None:
        see = see & ((qp - key).abs() < window)
    if prefix is not None:
        see = see & ((qp >= prefix) | (key <= qp))
    for h in range(H):
        kk, vv = k[:, h // (H // hkv)].double(), v[:, h // (H // hkv)].double()
        t = scale * (q[:, h].double() @ kk.T)
        if cap:
            t = cap * torch.tanh(t / cap)
        t = torch.where(see, t, -math.inf)
        p = torch.softmax(t, dim=-1)  # a row that sees nothing: NaN
        # Keys that a row does not see have no part in its sums.
        vz = torch.where(see.any(dim=0).view(-1, 1), vv, 0.0)
        out[:, h] = p @ vz
        mag[:, h] = p @ vz.abs()
    return out, mag
