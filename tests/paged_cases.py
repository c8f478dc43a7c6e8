"""Pools and batches of a paged cache for the tests, and what its operators compute, in 64 bits."""
import math

import torch

from polarquant_amd.paged import PageBatch, PagePool
from polarquant_amd.quantize import quantize_and_pack_nbit

PAGE = 128
F64 = torch.float64


class Cache:
    """Sequences of kv[b] tokens, the last new[b] of them a call's, the first sealed[b] pages sealed, over pages in no order; what no sequence holds is NaN
    (rows) or noise (codes).  `keys[b]`, `values[b]`: [Nk, kv, 128] in 64 bits, as the cache holds them."""

    def __init__(self, gpu, kv, new, sealed, N, Nk, dtype, rbits=4, tbits=4, packed=False, seed=0, spare=3, extra_rows=0, key_scale=1.0, wide=0):
        g = torch.Generator(device=gpu).manual_seed(seed)
        self.kv, self.new, self.sealed, self.N, self.Nk, self.dtype, self.gpu = kv, new, sealed, N, Nk, dtype, gpu
        B, held = len(kv), [-(-n // PAGE) for n in kv]
        W, Wo = max(max(held), 1) + wide, max(max(h - s for h, s in zip(held, sealed)), 1) + wide
        self.pages = torch.full((B, W), -1, dtype=torch.int32, device=gpu)
        self.open_pages = torch.full((B, Wo), -1, dtype=torch.int32, device=gpu)
        n_pages, n_open = sum(held) + spare, sum(h - s for h, s in zip(held, sealed)) + spare
        order, order_open = torch.randperm(n_pages, generator=g, device=gpu).int(), torch.randperm(n_open, generator=g, device=gpu).int()
        nan = float("nan")
        # (a stride between pages and heads of their own)
        keys = torch.full((n_open, Nk + 1, PAGE, 128), nan, dtype=dtype, device=gpu)[:, :Nk]
        values = torch.full((n_pages, Nk, PAGE, 128), nan, dtype=dtype, device=gpu)
        codes = torch.randint(0, 255, (n_pages, Nk, PAGE, 48 if packed else 64), generator=g, device=gpu, dtype=torch.uint8)
        meta = [torch.full((n_pages, Nk, 1, 64), nan, dtype=dtype, device=gpu) for _ in range(4)]
        self.keys, self.values, self.raw = [], [], []
        at = at_open = 0
        for b in range(B):
            k = torch.randn(Nk, kv[b], 128, generator=g, device=gpu).mul_(key_scale).to(dtype)
            v = torch.randn(Nk, kv[b], 128, generator=g, device=gpu).to(dtype)
            self.raw.append(k)
            self.pages[b, :held[b]] = order[at:at + held[b]]
            self.open_pages[b, :held[b] - sealed[b]] = order_open[at_open:at_open + held[b] - sealed[b]]
            at, at_open = at + held[b], at_open + held[b] - sealed[b]
            n = sealed[b] * PAGE
            exact = k.to(F64)
            if n:
                got = quantize_and_pack_nbit(k[None, :, :n].contiguous(), rbits, tbits, packed=packed)
                to = self.pages[b, :sealed[b]].long()
                for whole, part in zip([codes, *meta], got):
                    whole[to] = part[0].transpose(0, 1)
                exact[:, :n] = dequantized(got, rbits, tbits, packed)[0]
            for j in range(held[b]):
                m = min(PAGE, kv[b] - j * PAGE)
                values[self.pages[b, j].item(), :, :m] = v[:, j * PAGE:j * PAGE + m]
                if j >= sealed[b]:
                    keys[self.open_pages[b, j - sealed[b]].item(), :, :m] = k[:, j * PAGE:j * PAGE + m]
            self.keys.append(exact)
            self.values.append(v.to(F64))
        self.q_start = torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32, device=gpu)
        self.T = sum(new) + extra_rows
        self.q = torch.randn(max(self.T, 1), N, 128, generator=g, device=gpu).to(dtype)
        self.pool = PagePool(keys, values, codes, *meta, rbits=rbits, tbits=tbits)
        self.batch = self.batch_of()
        self.mask = None

    def batch_of(self, pages=None, open_pages=None, value_pages=None):
        def ints(v):
            return torch.tensor(v, dtype=torch.int32, device=self.gpu)
        return PageBatch(self.q_start, ints(self.kv), ints(self.sealed), self.pages if pages is None else pages, self.open_pages if open_pages is None else open_pages,
                         max(max(self.new), 1), max(max(self.kv), 1), value_pages)

    def rows(self):
        """(sequence, KV head, rows of q [n, rep, 128] in 64 bits, seen [n, kv]) of every sequence and KV head with new tokens."""
        rep = self.N // self.Nk
        for b, n in enumerate(self.new):
            if not n:
                continue
            first, kv = int(self.q_start[b]), self.kv[b]
            seen = torch.arange(kv, device=self.gpu) <= torch.arange(kv - n, kv, device=self.gpu)[:, None]
            if self.mask is not None:
                seen = seen & (self.mask[b, :kv] != 0)
            for h in range(self.Nk):
                yield b, h, slice(first, first + n), self.q[first:first + n, h * rep:(h + 1) * rep].to(F64), seen

    def attention(self, scale=None, gone=()):
        """-> (out, bound, lse, its bound): [T, N, 128], [T, N]; `gone`: (sequence, page) that do not exist.  Rows of no sequence are NaN.

        The bound, with u half a step of the dtype: a sealed key's cos and sin are rounded to float16 (2^-11 of them) and so is their product with the
        radius; the hardware's cos and sin, the angle in float32 and the sums of products add less than 3e-5.  So a score is off by at most
        d = scale |q| |k| (2^-10 + 3e-5), or 3e-5 for rows; a weight by exp(2 d) with the sum it is divided by, by u for its own rounding and n 2^-23 for the sums; the
        result is rounded once."""
        scale = 128 ** -0.5 if scale is None else scale
        u, rep = torch.finfo(self.dtype).eps / 2, self.N // self.Nk
        out = torch.full((self.T, self.N, 128), float("nan"), dtype=F64, device=self.gpu)
        tol, lse = torch.zeros_like(out), torch.full((self.T, self.N), float("nan"), dtype=F64, device=self.gpu)
        lse_tol = torch.zeros_like(lse)
        for b, h, at, q, seen in self.rows():
            k, v, n = self.keys[b][h], self.values[b][h], self.kv[b]
            seen = seen.clone()
            for s, p in gone:
                if s == b:
                    seen[:, p * PAGE:(p + 1) * PAGE] = False
            z = (torch.matmul(q.reshape(-1, 128), k.t().contiguous()) * scale).reshape(-1, rep, n).masked_fill(~seen[:, None], -math.inf)
            p = torch.softmax(z, -1).nan_to_num(0.0)
            heads = slice(h * rep, (h + 1) * rep)
            y = torch.matmul(p, torch.where(seen.any(0)[:, None], v, 0.0))
            off = torch.full((n,), 3e-5, dtype=F64, device=self.gpu)
            off[:self.sealed[b] * PAGE] += 2.0 ** -10
            d = abs(scale) * q.norm(dim=-1) * (k.norm(dim=-1) * off).amax()
            out[at, heads] = y
            tol[at, heads] = torch.matmul(p, v.abs()) * (torch.expm1(2 * d) + u + n * 2.0 ** -23)[..., None] + u * y.abs() + 1e-7
            lse[at, heads] = torch.logsumexp(z, -1)
            lse_tol[at, heads] = d + n * 2.0 ** -23 + 1e-5 + lse[at, heads].abs().nan_to_num(posinf=0.0) * 2.0 ** -22
        return out, tol, lse, lse_tol

    def page_weights(self, lse, W, scale=None):
        """-> (weights, bound) [B, Nk, W]: a sealed key is left with 2^-16 (bfloat16) or 2^-21 (float16) of itself by its two parts, 1e-5 covers cos and sin and
        the sums of products, n 2^-23 the sum of n weights."""
        scale = 128 ** -0.5 if scale is None else scale
        rep, left = self.N // self.Nk, 2.0 ** -16 if self.dtype == torch.bfloat16 else 2.0 ** -21
        out = torch.zeros(len(self.kv), self.Nk, W, dtype=F64, device=self.gpu)
        tol = torch.zeros_like(out)
        for b, h, at, q, seen in self.rows():
            n = self.kv[b]
            z = (torch.matmul(q.reshape(-1, 128), self.keys[b][h].t().contiguous()) * scale).reshape(-1, rep, n).masked_fill(~seen[:, None], -math.inf)
            log_sum = lse[at, h * rep:(h + 1) * rep, None].to(F64)
            p = torch.where(torch.isfinite(log_sum), torch.exp(z - log_sum), 0.0).sum((0, 1))
            d = float(abs(scale) * q.norm(dim=-1).amax() * self.keys[b][h].norm(dim=-1).amax()) * (left + 1e-5) + 128 * q.shape[0] * rep * 2.0 ** -23 + 1e-5
            for j in range(-(-n // PAGE)):
                out[b, h, j] = p[j * PAGE:(j + 1) * PAGE].sum()
                tol[b, h, j] = out[b, h, j] * math.expm1(d) + 1e-30
        return out, tol


def dequantized(parts, rbits, tbits, packed=False):
    """Codes [B, Nk, groups, 128, 64] and constants -> keys [B, Nk, groups * 128, 128] in 64 bits."""
    codes, rscale, rmn, tscale, tmn = parts
    if packed:
        from polarquant_amd.quantize import convert_codes6
        codes = convert_codes6(codes, False)
    theta, rho = (codes & (2 ** tbits - 1)).to(F64), (codes >> tbits).to(F64)
    phi, r = tscale.to(F64) * (theta + 0.5) + tmn.to(F64), rscale.to(F64) * (rho + 0.5) + rmn.to(F64)
    return torch.cat([r * phi.cos(), r * phi.sin()], -1).flatten(2, 3)


def evicted(weights, pages, n_sealed, kv_len, keep, sinks):
    """What evict_pages leaves, from lists."""
    W, out = len(pages[0]), []
    for w, row, n, kv in zip(weights, pages, n_sealed, kv_len):
        total = torch.tensor(w, dtype=F64).sum(0).float().tolist()
        always = list(range(min(sinks, n)))
        stay = list(range(n)) if n <= keep else sorted(always + sorted(range(len(always), n), key=lambda j: (-total[j], j))[:keep - len(always)])
        gone = [j for j in range(n) if j not in set(stay)]
        left = stay + [j for j in range(n, W) if row[j] >= 0]
        out.append(([row[j] for j in left] + [-1] * (W - len(left)), len(stay), kv - PAGE * len(gone),
                    [[head[j] for j in left] + [0.0] * (W - len(left)) for head in w], [row[j] for j in gone] + [-1] * (W - len(gone))))
    return [list(x) for x in zip(*out)]
