"""The 4-bit cache and attention over it in 64 bits, from the definition, and the bound that the kernels' roundings give."""

from __future__ import annotations

import math

import torch

FP4 = torch.float4_e2m1fn_x2
E8M0 = torch.float8_e8m0fnu
BLOCK = 32
VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def encode(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """[..., dim] -> (codes [..., dim], exponent bytes [..., dim / 32]), by trying every value and every exponent's limit."""

    b = x.double().unflatten(-1, (-1, BLOCK))
    amax = b.abs().amax(-1)
    bad = ~torch.isfinite(amax)
    amax = torch.where(bad, 0.0, amax)
    limits = 7.0 * torch.exp2(torch.arange(-126, 126, dtype=torch.float64))
    e = torch.searchsorted(limits, amax) - 126  # the first limit that is not below amax
    units = torch.where(bad[..., None], 0.0, b) / torch.exp2(e.double())[..., None]
    grid = torch.tensor(VALUES, dtype=torch.float64)
    far = (units.abs()[..., None] - grid).abs()
    # nearest, of two as near the even code
    codes = (far * 4 + torch.tensor([0, 1] * 4) * 1e-9 * (far == far.amin(-1, keepdim=True))).argmin(-1)
    codes = codes + 8 * torch.signbit(units)
    return codes.flatten(-2).to(torch.uint8), torch.where(bad, 255, e + 127).to(torch.uint8)


def pack(codes: torch.Tensor) -> torch.Tensor:
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def decode(payload: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """Payload and exponents (any dtype of one byte) -> fp64 values."""

    p = payload.cpu().view(torch.uint8)
    codes = torch.stack([p & 15, p >> 4], dim=-1).flatten(-2).long()
    grid = torch.tensor(VALUES + [-v for v in VALUES], dtype=torch.float64)
    e = scales.cpu().view(torch.uint8)
    scale = torch.where(e == 255, math.nan, torch.exp2(e.double() - 127))
    return (grid[codes].unflatten(-1, (-1, BLOCK)) * scale[..., None]).flatten(-2)


def quantized(x: torch.Tensor, device="cuda") -> tuple[torch.Tensor, torch.Tensor]:
    codes, e = encode(x.cpu())
    return pack(codes).to(device).view(FP4), e.to(device).view(E8M0)


def empty_cache(shape, device="cuda", fill=0x55, exponent=127):
    """A pool [blocks, page, heads, dim] of 4-bit K or V with something in it."""

    payload = torch.full((*shape[:-1], shape[-1] // 2), fill, dtype=torch.uint8, device=device).view(FP4)
    scales = torch.full((*shape[:-1], shape[-1] // BLOCK), exponent, dtype=torch.uint8, device=device).view(E8M0)
    return payload, scales


def attend(q, k, v, scale, visible, weight=2.0 ** -8):
    """q [rows, dim], k and v [keys, dim] in 64 bits, visible [rows, keys] -> (output, bound on the kernel's error).

    The bound counts, per row, with w the weights and A = sum w |v|:
      weight A        weights times exponents rounded: 2^-8 to bf16, 2^-11 to float16, 2^-16 to two bf16 numbers;
      2 ds A          weights off because scores are off by up to ds (numerator and denominator);
      2^-18 A         fp32 sums of weights and outputs, parts joined (a few hundred roundings of 2^-24);
      2^-126 sum (|v| + 6)  weights (the largest is 1), and weights times exponents, below the smallest normal number
                      are 0: a weight less than 2^-126 off times v, a product less than 2^-126 off times at most 6;
    ds: fp32 sums of up to 128 exact products and a few roundings (each 2^-24 of what is summed), the exponent's argument
    and the exponential (2^-22 of the argument's magnitude, and 2^-22).  The output's own rounding is the caller's.
    """

    logits = (q @ k.t()) * scale
    sums = (q.abs() @ k.abs().t()) * abs(scale)
    low = torch.where(visible, logits, -math.inf)
    top = low.amax(1, keepdim=True)
    w = torch.where(visible, torch.exp(low - torch.where(torch.isfinite(top), top, 0.0)), 0.0)
    total = w.sum(1, keepdim=True)
    w = w / torch.where(total > 0, total, 1.0)
    ds = 132 * 2.0 ** -24 * sums + 2.0 ** -22 * (2 * sums + 1)
    ds = torch.where(visible, ds, 0.0).amax(1, keepdim=True)
    at = w @ v.abs()
    lost = 2.0 ** -126 * (visible.double() @ (v.abs() + 6.0))
    if weight == 2.0 ** -11:  # float16 weights, 2^7 times exp(score - max), end at half of 2^-24
        lost = lost + 2.0 ** -32 * (visible.double() @ v.abs())
    return w @ v, (weight + 2 * ds + 2.0 ** -18) * at + lost


def check(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, label="") -> None:
    """|got - want| <= bound + the rounding of what was computed to got's type."""

    g = got.double().cpu()
    half = torch.finfo(got.dtype).eps / 2
    limit = bound + half * (want.abs() + bound) + torch.finfo(got.dtype).tiny
    bad = ~((g - want).abs() <= limit)
    worst = float(((g - want).abs() / limit).nan_to_num(0).max()) if g.numel() else 0.0
    print(f"[{label}] worst error {worst:.3f} of the bound", flush=True)
    assert torch.isfinite(g).all(), f"{label}: not finite"
    assert not bad.any(), (f"{label}: {int(bad.sum())} of {bad.numel()} values beyond the bound, worst {worst:.3f} of it: "
                           f"{g[bad][:4].tolist()} for {want[bad][:4].tolist()}, bound {limit[bad][:4].tolist()}")


class Pool:
    """A 4-bit cache of quantised random tokens in scattered pages, for sequences of given lengths."""

    def __init__(self, ctx, *, page, kv_heads, dim, seed, spare=3, spread=True):
        g = torch.Generator().manual_seed(seed)
        self.ctx, self.page = list(ctx), page
        need = [-(-n // page) for n in self.ctx]
        blocks = sum(need) + spare
        self.width = max(max(need, default=0), 1)
        k = torch.randn(blocks, page, kv_heads, dim, generator=g)
        v = torch.randn(blocks, page, kv_heads, dim, generator=g)
        if spread:  # exponents that differ from block to block
            k = k * torch.exp2(torch.randint(-2, 3, (blocks, page, kv_heads, dim // BLOCK), generator=g).float()).repeat_interleave(BLOCK, -1)
            v = v * torch.exp2(torch.randint(-4, 5, (blocks, page, kv_heads, dim // BLOCK), generator=g).float()).repeat_interleave(BLOCK, -1)
        self.kc, self.ks = quantized(k)
        self.vc, self.vs = quantized(v)
        order = torch.randperm(blocks, generator=g).to(torch.int32)
        tables = torch.full((len(self.ctx), self.width), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            tables[i, :n] = order[at:at + n]
            at += n
        self.tables = tables.cuda()
        self.lens = torch.tensor(self.ctx, dtype=torch.int32, device="cuda")

    def rows(self, i, n=None):
        """Sequence i's keys and values in 64 bits, [tokens, heads, dim]; tokens in missing pages are left out (with their places)."""

        n = self.ctx[i] if n is None else n
        table = self.tables[i].cpu().tolist()
        blocks = self.kc.shape[0]
        keep = [t for t in range(n) if 0 <= table[t // self.page] < blocks]
        b = torch.tensor([table[t // self.page] for t in keep], dtype=torch.long)
        r = torch.tensor([t % self.page for t in keep], dtype=torch.long)
        pick = lambda c: c.view(torch.uint8).cpu()[b, r]  # noqa: E731
        return decode(pick(self.kc), pick(self.ks)), decode(pick(self.vc), pick(self.vs)), torch.tensor(keep, dtype=torch.long)


def decode_reference(pool: Pool, q, scale, limit=None):
    """Expected decode output and bound, [batch, heads, dim]."""

    weight = 2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -16
    q = q.double().cpu()
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for i in range(q.shape[0]):
        n = pool.ctx[i] if limit is None else min(pool.ctx[i], limit)
        k, v, keep = pool.rows(i, max(n, 0))
        if keep.numel() == 0:
            continue
        group = q.shape[1] // k.shape[1]
        for h in range(k.shape[1]):
            rows = slice(h * group, (h + 1) * group)
            out[i, rows], bound[i, rows] = attend(q[i, rows], k[:, h], v[:, h], scale, torch.ones(group, keep.numel(), dtype=torch.bool), weight)
    return out, bound


def chunk_reference(pool: Pool, q, cu, scale):
    """Expected chunk output and bound, with q's rows (zeros outside the sequences)."""

    weight = 2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -11
    q = q.double().cpu()
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for i, (a, b) in enumerate(zip(cu, cu[1:])):
        k, v, keep = pool.rows(i)
        n, m = b - a, pool.ctx[i]
        group = q.shape[1] // k.shape[1]
        for h in range(k.shape[1]):
            for j in range(h * group, (h + 1) * group):
                seen = keep[None, :] <= (m - n + torch.arange(n))[:, None]
                out[a:b, j], bound[a:b, j] = attend(q[a:b, j], k[:, h], v[:, h], scale, seen, weight)
    return out, bound
