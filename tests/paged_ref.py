"""Plain 64-bit forms of the paged-cache operators, and how far the kernels may be from them."""
import math

import torch

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # half a rounding step, relative


class Batch:
    """Sequences with q_lens[i] new tokens and kv_lens[i] keys (the new ones included) over a pool of pages in random order.
    Everything that belongs to no sequence - free pages, slots past the end, table entries past the last page - is poison."""

    def __init__(self, q_lens, kv_lens, nqh, nkv, hd, page, dtype, seed=0, spare_rows=0, poison=True, values=1.0):
        g = torch.Generator().manual_seed(seed)
        self.q_lens, self.kv_lens, self.nqh, self.nkv, self.hd, self.page, self.dtype = q_lens, kv_lens, nqh, nkv, hd, page, dtype
        self.total = sum(q_lens) + spare_rows
        need = [-(-n // page) for n in kv_lens]
        self.n_pages = sum(need) + 3
        order = torch.randperm(self.n_pages, generator=g)[:sum(need)].tolist()
        bad = float("nan") if poison else 0.0
        self.k = torch.full((self.n_pages, page, nkv, hd), bad, dtype=dtype)
        self.v = torch.full((self.n_pages, page, nkv, hd), bad, dtype=dtype)
        self.table = torch.full((len(kv_lens), max(max(need), 1)), -7 if poison else 0, dtype=torch.int32)
        self.keys, self.vals, at = [], [], 0
        for s, n in enumerate(kv_lens):
            pages = order[at:at + need[s]]
            at += need[s]
            self.table[s, :need[s]] = torch.tensor(pages, dtype=torch.int32)
            ks = (torch.randn(n, nkv, hd, generator=g)).to(dtype)
            vs = (values * torch.randn(n, nkv, hd, generator=g)).to(dtype)
            for j, pg in enumerate(pages):
                m = min(page, n - j * page)
                self.k[pg, :m], self.v[pg, :m] = ks[j * page:j * page + m], vs[j * page:j * page + m]
            self.keys.append(ks.cuda()), self.vals.append(vs.cuda())
        self.q = torch.randn(self.total, nqh * hd, generator=g).to(dtype).cuda()
        cu = [0]
        for n in q_lens:
            cu.append(cu[-1] + n)
        self.cu = torch.tensor(cu, dtype=torch.int32).cuda()
        self.kv_len = torch.tensor(kv_lens, dtype=torch.int32).cuda()
        self.k, self.v, self.table = self.k.cuda(), self.v.cuda(), self.table.cuda()
        self.max_q, self.max_kv = max(q_lens), max(kv_lens)

    def rows(self, s):
        a = sum(self.q_lens[:s])
        return slice(a, a + self.q_lens[s])


def attention(q, k, v, scale, window, p_dtype, out_dtype):
    """q (n, nqh, hd), k and v (t, nkv, hd): row i is position t - n + i.  Returns the output in 64 bits (n, nqh, hd) and the
    bound on what a kernel's may differ by, which counts: the probabilities rounded to p_dtype (half a step of each, and half a
    subnormal step), scores and sums in f32 (a step of 2^-23 per addition, truncation allowed), the exponential (2^-21 and the
    rounding of its argument), the output rounded to out_dtype."""
    n, nqh, hd = q.shape
    t, nkv = k.shape[0], k.shape[1]
    out = torch.zeros(n, nqh, hd, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    pos = torch.arange(t - n, t, device=q.device)[:, None]
    key = torch.arange(t, device=q.device)[None]
    seen = key <= pos
    if window:
        seen &= key > pos - window
    some = seen.any(dim=1)
    if not some.any():
        return out, tol
    for h in range(nqh):
        kd, vd, qd = k[:, h // (nqh // nkv)].double(), v[:, h // (nqh // nkv)].double(), q[:, h].double()
        vd = torch.where(torch.isfinite(vd), vd, 0.0) if not torch.isfinite(vd).all() else vd
        x = (qd @ kd.T) * scale
        x = torch.where(seen, x, float("-inf"))
        m = x.amax(dim=1, keepdim=True)
        m = torch.where(torch.isfinite(m), m, 0.0)
        p = torch.exp(x - m)
        total = p.sum(dim=1, keepdim=True).clamp(min=1e-300)
        o = p @ vd / total
        size = p @ vd.abs() / total
        score = (hd + 2) * 2.0 ** -23 * scale * torch.where(seen, qd.abs() @ kd.abs().T, 0.0).amax(dim=1, keepdim=True)
        arg = 2.0 ** -23 * torch.where(seen, (x - m).abs(), 0.0).amax(dim=1, keepdim=True).clamp(max=40.0)
        rel = HALF[p_dtype] + 2 * (score + arg + 2.0 ** -21) + (seen.sum(dim=1, keepdim=True) + 64) * 2.0 ** -23
        small = 2.0 ** -25 * seen.sum(dim=1, keepdim=True) * vd.abs().max() / total if p_dtype == torch.float16 else 0.0
        e = size * rel + small
        out[:, h] = torch.where(some[:, None], o, 0.0)
        tol[:, h] = torch.where(some[:, None], e + HALF[out_dtype] * (o.abs() + e) + (2.0 ** -25 if out_dtype == torch.float16 else 0.0), 0.0)
    return out, tol


def expect(b, scale, window, out_dtype, packed=False):
    """The 64-bit output and bound of a whole batch (rows of no sequence: nan)."""
    out = torch.full((b.total, b.nqh, b.hd), float("nan"), dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    for s, n in enumerate(b.q_lens):
        if n:
            r = b.rows(s)
            out[r], tol[r] = attention(b.q[r].view(n, b.nqh, b.hd), b.keys[s], b.vals[s], scale, window, b.dtype, out_dtype)
    return out, tol


def near(got, want, tol, what=""):
    got = got.double().view(want.shape)
    rows = ~torch.isnan(want)
    assert torch.isfinite(got[rows]).all(), f"{what}: not finite"
    over = (got - want).abs()[rows] - tol[rows]
    assert over.numel() == 0 or over.max() <= 0, f"{what}: {int((over > 0).sum())} of {over.numel()} off, by up to {float(over.max()):.3e} more than {float(tol[rows].max()):.3e}"


def rotate(x, pos, rot, theta):
    """NeoX pairs of the first `rot` elements of x (n, heads, hd), in 64 bits."""
    x = x.double().clone()
    half = rot // 2
    angle = pos.double()[:, None] * torch.exp(-2.0 * math.log(theta) / max(rot, 1) * torch.arange(half, device=x.device).double())
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x[..., :half].clone(), x[..., half:rot].clone()
    x[..., :half], x[..., half:rot] = a * c - b * s, a * s + b * c
    return x
