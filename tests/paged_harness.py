"""Test infrastructure of the paged-cache tests: random steps, and the operators' definitions in 64 bits on the CPU."""
import math

import torch


def unit(dtype):
    """Largest relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


class Case:
    """Sequences (new rows, length afterwards) over a cache with shuffled pages, everything on the CPU."""

    def __init__(self, seqs, nq, nkv, hn, ps, dtype, pad=0, seed=0, spare_pages=2, garbage=None):
        g = torch.Generator().manual_seed(seed)
        self.seqs, self.nq, self.nkv, self.hn, self.ps, self.dtype = seqs, nq, nkv, hn, ps, dtype
        need = [max(1, -(-max(l, 0) // ps)) for _, l in seqs]
        self.num_pages = sum(need) + spare_pages
        perm = torch.randperm(self.num_pages, generator=g).to(torch.int32)
        self.block_table = torch.full((len(seqs), max(need)), -1, dtype=torch.int32)  # -1 behind a sequence's last page
        at = 0
        for i, n in enumerate(need):
            self.block_table[i, :n] = perm[at:at + n]
            at += n
        self.cu = torch.tensor([0] + [n for n, _ in seqs]).cumsum(0).to(torch.int32)
        self.lens = torch.tensor([l for _, l in seqs], dtype=torch.int32)
        self.rows = int(self.cu[-1]) + pad
        shape = (self.num_pages, nkv, ps, hn)
        self.k_cache = torch.randn(shape, generator=g).to(dtype)
        self.v_cache = torch.randn(shape, generator=g).to(dtype)
        if garbage is not None:  # what no row may see: slots behind the sequences' ends and pages of no sequence
            seen = torch.zeros(self.num_pages, ps, dtype=torch.bool)
            for i, (_, l) in enumerate(seqs):
                for p in range(max(l, 0)):
                    seen[self.block_table[i, p // ps], p % ps] = True
            hide = (~seen)[:, None, :, None].expand(shape)
            self.k_cache[hide] = garbage
            self.v_cache[hide] = garbage
        self.q = (torch.randn(self.rows, nq, hn, generator=g) * 1.5).to(dtype)
        self.k = torch.randn(self.rows, nkv, hn, generator=g).to(dtype)
        self.v = torch.randn(self.rows, nkv, hn, generator=g).to(dtype)
        self.scale = 1.0 / math.sqrt(hn)

    @property
    def max_new(self):
        return max(n for n, _ in self.seqs)

    @property
    def max_kv(self):
        return max(0, max(l for _, l in self.seqs))

    def step(self, device="cuda", **kw):
        from multimodal_amd.kv_cache import PagedStep
        kw.setdefault("max_new", self.max_new)
        kw.setdefault("max_kv", self.max_kv)
        return PagedStep(self.block_table.to(device), self.cu.to(device), self.lens.to(device), **kw)

    def kv(self, device="cuda"):
        from multimodal_amd.kv_cache import PagedKV
        return PagedKV(self.k_cache.to(device), self.v_cache.to(device))

    def keys_values(self, i):
        """[len, nkv, hn] of sequence i in 64 bits, and the validity of each key's page."""
        l = max(int(self.lens[i]), 0)
        pos = torch.arange(l)
        page = self.block_table[i].long()[pos // self.ps]
        ok = (page >= 0) & (page < self.num_pages)
        page = torch.where(ok, page, torch.zeros_like(page))
        return self.k_cache[page, :, pos % self.ps].double(), self.v_cache[page, :, pos % self.ps].double(), ok


def attention_oracle(c):
    """(out, lse, tol_out, tol_lse) in 64 bits; NaN where a row sees a page the cache does not have.  Tolerances, with u the
    rounding of the dtype: the output is rounded once and the probabilities once (u each, relative to softmax |v|); a score is a
    sum of hn fp32 products (hn 2^-24 of the sum of their magnitudes) scaled and shifted in fp32 (two roundings of a number
    up to |s| + |lse|), which moves p by that much relative, and exp2, log2 and the division are good to 2^-21; the sum of the
    probabilities adds len 2^-24.  Numerator and denominator both carry the score's error."""
    out = torch.zeros(c.rows, c.nq, c.hn, dtype=torch.float64)
    lse = torch.full((c.rows, c.nq), float("nan"), dtype=torch.float64)
    t_out, t_lse = torch.zeros(c.rows, c.nq, c.hn, dtype=torch.float64), torch.zeros(c.rows, c.nq, dtype=torch.float64)
    u = unit(c.dtype)
    for i, (n, l) in enumerate(c.seqs):
        k, v, ok = c.keys_values(i)
        for j in range(n):
            row, p = int(c.cu[i]) + j, l - n + j
            if p < 0:
                lse[row] = -math.inf
                continue
            for h in range(c.nq):
                kh = h // (c.nq // c.nkv)
                kk, vv = k[:p + 1, kh], v[:p + 1, kh]
                q = c.q[row, h].double()
                s = (kk @ q) * c.scale
                if not bool(ok[:p + 1].all()):
                    s = s * float("nan")
                mag = (kk.abs() @ q.abs()).max() * c.scale
                z = torch.logsumexp(s, 0)
                w = torch.exp(s - z)
                out[row, h], lse[row, h] = w @ vv, z
                ds = c.hn * 2.0 ** -24 * mag + 2.0 ** -22 * (s.abs().max() + z.abs()) + 2.0 ** -21
                t_out[row, h] = 1.01 * (2 * u + 2 * ds + (p + 1) * 2.0 ** -24) * (w @ vv.abs()) + 1e-30
                t_lse[row, h] = ds + (p + 1) * 2.0 ** -24 + 2.0 ** -22 * z.abs()
    return out, lse, t_out, t_lse


def check_attention(c, out, lse, what=""):
    """Rows of sequences against the oracle; NaN and infinities must be where the oracle has them."""
    eo, el, to, tl = attention_oracle(c)
    n = int(c.cu[-1])
    out, lse = out[:n].double().cpu(), lse[:n].double().cpu()
    eo, el, to, tl = eo[:n], el[:n], to[:n], tl[:n]
    assert torch.equal(torch.isnan(out), torch.isnan(eo)), f"{what}: NaN in other places than the definition's"
    inf = torch.isinf(eo)
    assert torch.equal(out[inf], eo[inf]), f"{what}: infinities"
    fin = torch.isfinite(eo)
    excess = ((out - eo).abs() - to)[fin]
    assert excess.numel() == 0 or excess.max() <= 0, f"{what}: output off by {excess.max()} more than the tolerance"
    # lse of a row with NaN is NaN, of an empty row -inf
    assert torch.equal(torch.isnan(lse), torch.isnan(el)) and torch.equal(torch.isinf(lse), torch.isinf(el)), f"{what}: lse"
    fin = torch.isfinite(el)
    assert not fin.any() or ((lse - el).abs() - tl)[fin].max() <= 0, f"{what}: lse off"


def append_oracle(c, cos=None, sin=None):
    """(q_out, k_cache, v_cache, tolerances of the first two): one rounding to the dtype, two products and a sum in fp32."""
    u = unit(c.dtype)
    kc, vc = c.k_cache.double(), c.v_cache.double()
    qo = torch.zeros(c.rows, c.nq, c.hn, dtype=torch.float64)
    tq, tk = torch.zeros_like(qo), torch.zeros_like(kc)

    def rot(x, p):
        x = x.double()
        if cos is None:
            return x, torch.zeros_like(x)
        d = cos.size(-1)
        a, b = x[..., :d // 2], x[..., d // 2:d]
        cc, ss = cos[p].double(), sin[p].double()
        r = torch.cat((-b, a), -1)
        y = x.clone()
        y[..., :d] = x[..., :d] * cc + r * ss
        t = torch.zeros_like(x)
        t[..., :d] = y[..., :d].abs() * u + ((x[..., :d] * cc).abs() + (r * ss).abs()) * 2.0 ** -22
        return y, t

    for i, (n, l) in enumerate(c.seqs):
        for j in range(n):
            row, p = int(c.cu[i]) + j, l - n + j
            page = int(c.block_table[i, p // c.ps]) if 0 <= p < c.block_table.size(1) * c.ps else -1
            if p < 0 or not 0 <= page < c.num_pages or (cos is not None and p >= cos.size(0)):
                qo[row] = float("nan")
                continue
            qo[row], tq[row] = rot(c.q[row], p)
            kc[page, :, p % c.ps], tk[page, :, p % c.ps] = rot(c.k[row], p)
            vc[page, :, p % c.ps] = c.v[row].double()
    return qo, kc, vc, tq, tk


def tables(positions, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + 99)
    inv = 1.0 / (10000.0 ** (torch.arange(0, d, 2, dtype=torch.float64) / d))
    ang = torch.arange(positions, dtype=torch.float64)[:, None] * inv
    # the two halves of a rotary table are equal; a perturbed second half shows that each half reads its own column
    ang = torch.cat((ang, ang + 0.1 * torch.rand(1, generator=g).double()), dim=1)
    return ang.cos().to(dtype), ang.sin().to(dtype)
