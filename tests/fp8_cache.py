"""A cache in 8 bits restated in plain torch on the CPU: what holds a number, what an append leaves, what attention gives.

A block of 16 positions of a head has an exponent e, the smallest in [-64, 119] with (largest finite magnitude) 2^-e <= 448,
and a number x is held as the e4m3 number nearest to x 2^-e (ties to even). Nothing here calls the library."""
import math

import torch

PAGE, BLOCK = 64, 16
E_MIN, E_MAX = -64, 119
F8 = torch.float8_e4m3fn


def exponent_of(x: torch.Tensor) -> int:
    """x: the numbers of one block of one head."""
    x = x.double()
    x = x[torch.isfinite(x)].abs()
    big = float(x.max()) if x.numel() else 0.0
    if big == 0.0:
        return E_MIN
    e = math.ceil(math.log2(big / 448.0))
    while big * 2.0 ** -e > 448.0:          # log2 is rounded: settle it by the definition
        e += 1
    while big * 2.0 ** -(e - 1) <= 448.0:
        e -= 1
    return min(max(e, E_MIN), E_MAX)


def to_codes(x: torch.Tensor, e: int) -> torch.Tensor:
    """float32 numbers of a block as e4m3; what is not finite becomes NaN, what is above 448 * 2^119 that number."""
    y = (x.double() * 2.0 ** -e).float()
    y = torch.where(torch.isfinite(x), y.clamp(-448.0, 448.0), torch.full_like(y, math.nan))
    return y.to(F8)


def rotate(x: torch.Tensor, table: torch.Tensor, rot: int) -> torch.Tensor:
    """x float32 [T, heads, hd], table float32 [T, rot / 2, 2] of (cos, sin): each product and each sum rounded to float32."""
    if rot == 0:
        return x
    c, s = table[:, None, :, 0], table[:, None, :, 1]
    a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., rot:]], -1)


class PlainCache:
    """Pages of codes and exponents with the sequences' tables, filled with what former owners may have left."""

    def __init__(self, lens, n_kv, hd, seed=0, nan_stale=False):
        """lens: the longest that each sequence gets."""
        g = torch.Generator().manual_seed(seed)
        n = len(lens)
        need = [(l + PAGE - 1) // PAGE for l in lens]
        self.n_pages = sum(need) + 4
        perm = torch.randperm(self.n_pages - 1, generator=g).tolist()
        self.slots = torch.randperm(n + 3, generator=g)[:n].tolist()
        self.table = torch.full((n + 3, max(need) + 1), self.n_pages - 1, dtype=torch.int32)
        for i, s in enumerate(self.slots):
            for p in range(need[i]):
                self.table[s, p] = perm.pop()
        self.n_kv, self.hd = n_kv, hd
        shape = (self.n_pages, n_kv, PAGE, hd)

        def stale():
            codes = torch.randint(0, 256, shape, generator=g, dtype=torch.int16).to(torch.uint8)
            if not nan_stale:
                codes[(codes & 0x7f) == 0x7f] = 0x31
            return codes.view(F8)

        self.k, self.v = stale(), stale()
        self.ke = torch.randint(-20, 20, shape[:2] + (4,), generator=g).to(torch.int8)
        self.ve = torch.randint(-20, 20, shape[:2] + (4,), generator=g).to(torch.int8)

    def where(self, i, pos):
        return int(self.table[self.slots[i], pos // PAGE]), pos % PAGE

    def append(self, i, start, keys, values):
        """Rotated float32 keys and values [m, n_kv, hd] of positions start, start + 1, ... of sequence i."""
        m = keys.shape[0]
        for b in range(start // BLOCK, (start + m - 1) // BLOCK + 1):
            lo, hi = max(start, b * BLOCK), min(start + m, b * BLOCK + BLOCK)
            page, row0 = self.where(i, b * BLOCK)
            lead = lo - b * BLOCK
            for codes, exps, x in ((self.k, self.ke, keys), (self.v, self.ve, values)):
                for h in range(self.n_kv):
                    new = x[lo - start:hi - start, h]
                    e = exponent_of(new)
                    if lead:
                        old = min(max(int(exps[page, h, row0 // BLOCK]), E_MIN), E_MAX)
                        e = max(e, old)
                        if e > old:
                            kept = codes[page, h, row0:row0 + lead].float()
                            codes[page, h, row0:row0 + lead] = to_codes(kept, e - old)
                    codes[page, h, row0 + lead:row0 + lead + hi - lo] = to_codes(new, e)
                    exps[page, h, row0 // BLOCK] = e

    def held(self, i, length):
        """Keys and values of sequence i as they are held, float64 [length, n_kv, hd]."""
        out = []
        for codes, exps in ((self.k, self.ke), (self.v, self.ve)):
            at = torch.arange(length)
            page = self.table[self.slots[i]].long()[at // PAGE]
            x = codes.view(torch.uint8)[page, :, at % PAGE].view(F8).double()
            out.append(x * 2.0 ** exps[page, :, at % PAGE // BLOCK].double()[..., None])
        return out

    def dev(self, device="cuda"):
        return self.k.to(device), self.v.to(device), self.ke.to(device), self.ve.to(device)


def attention(q, k, v, positions, scale, window):
    """q [T, n_q, hd] at absolute positions, k, v [L, n_kv, hd], all float64; window as the kernels take it. Returns the output
    and sum_j p_j |v_j|, which errors of the weights are relative to."""
    group = q.shape[1] // k.shape[1]
    out, size = torch.empty_like(q), torch.empty_like(q)
    for t, p in enumerate(positions):
        lo = max(0, p - window + 1) if window > 0 else p - p % -window if window < 0 else 0
        kk, vv = k[lo:p + 1].repeat_interleave(group, 1), v[lo:p + 1].repeat_interleave(group, 1)
        w = torch.softmax(torch.einsum("hd,jhd->hj", q[t], kk) * scale, -1)
        out[t] = torch.einsum("hj,jhd->hd", w, vv)
        size[t] = torch.einsum("hj,jhd->hd", w, vv.abs())
    return out, size
