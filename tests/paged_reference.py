"""Plain 64-bit forms of the paged operators (torch double), and batches to try them on."""
import math

import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # a rounding is off by at most this much of the value
LEAST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}     # ... or by this much, below the normal numbers


def rotate(x, pos, theta, w=None, eps=1e-5):
    """[rows, heads, dh] doubles: norm of every head weighted by w [heads, dh] (None: no norm), adjacent pairs turned."""
    dh = x.shape[-1]
    if w is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    a = pos.double()[:, None, None] * theta ** (-2.0 * torch.arange(dh // 2, dtype=torch.float64, device=x.device) / dh)
    e, o = x[..., 0::2], x[..., 1::2]
    return torch.stack([e * a.cos() - o * a.sin(), e * a.sin() + o * a.cos()], -1).flatten(-2)


def rotate_tolerance(x, pos, theta, w, eps, dt, ref):
    """One rounding of the result, plus the f32 steps in front of it.  A product of norm, weight and rotation: r is a sum of dh
    squares (its relative error at most (dh + 4) 2^-24, halved by the root, plus 2 ulp of rsqrtf and the divisions), n = x r w two
    roundings more, sin and cos are off by 2 ulp and the angle, reduced to [-pi, pi] from f64 into f32, by pi 2^-24; the two
    products and their sum round three times.  All relative to |n[2k]| + |n[2k+1]|: (dh / 2 + 20) 2^-24 covers it."""
    dh = x.shape[-1]
    n = x if w is None else x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    pair = (n[..., 0::2].abs() + n[..., 1::2].abs()).repeat_interleave(2, -1)
    f32 = (dh / 2 + 20) * 2.0 ** -24 * pair
    return HALF_STEP[dt] * (ref.abs() + f32) + f32 + LEAST[dt]


class Batch:
    """Sequences with n new tokens and kv slots, their pages shuffled; every slot and table entry that is not theirs holds
    something that must never show (NaN, a page far outside)."""

    def __init__(self, dev, dt, n, kv, nkvh, dh, ps, pad=0, seed=0, order="page_head_slot", index=torch.int32, spare=2, first=0, max_seq=0):
        g = torch.Generator().manual_seed(seed)
        self.n, self.kv, self.ps, self.nkvh, self.dh, self.dt, self.dev, self.max_seq = list(n), list(kv), ps, nkvh, dh, dt, dev, max_seq
        self.first = first
        self.nt = first + sum(n) + pad
        pages = [-(-l // ps) for l in kv]
        self.npages = sum(pages) + spare
        perm = torch.randperm(self.npages, generator=g)
        width = max(pages + [1]) + 1
        self.table = torch.full((len(kv), width), 0x7ffffff0, dtype=torch.int64)
        at = 0
        for i, c in enumerate(pages):
            self.table[i, :c] = perm[at: at + c]
            at += c
        self.spares = perm[at:].tolist()  # pages of nobody
        self.start = first + torch.tensor([sum(n[:i]) for i in range(len(n) + 1)])
        self.page_table, self.seq_start, self.kv_len = (t.to(torch.int32).to(dev).view(index) for t in (self.table, self.start, torch.tensor(kv)))
        shape = {"page_head_slot": (self.npages, nkvh, ps, dh), "page_slot_head": (self.npages, ps, nkvh, dh), "joint": (self.npages, 2, ps, nkvh, dh)}[order]
        if order == "joint":  # keys and values of a page side by side, slots in front of heads
            both = torch.full(shape, math.nan, dtype=dt, device=dev)
            self.k_pages, self.v_pages = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
        else:
            self.k_pages, self.v_pages = (torch.full(shape, math.nan, dtype=dt, device=dev) for _ in range(2))
            if order == "page_slot_head":
                self.k_pages, self.v_pages = self.k_pages.transpose(1, 2), self.v_pages.transpose(1, 2)

    def slots(self, i, lo, hi):
        """(page, slot) of sequence i's slots [lo, hi)."""
        s = torch.arange(lo, hi)
        return self.table[i, s // self.ps].to(self.dev), (s % self.ps).to(self.dev)

    def fill(self, g, std_k=1.0):
        """Random keys and values in every sequence's slots."""
        for i, l in enumerate(self.kv):
            if l:
                page, slot = self.slots(i, 0, l)
                self.k_pages[page, :, slot] = (std_k * torch.randn(l, self.nkvh, self.dh, generator=g, device=self.dev)).to(self.dt)
                self.v_pages[page, :, slot] = torch.randn(l, self.nkvh, self.dh, generator=g, device=self.dev).to(self.dt)

    def descriptor(self, pkg):
        return pkg.PagedBatch(self.page_table, self.seq_start, self.kv_len, self.max_seq)


def attention(b, q, causal, scale, skip=()):
    """(o, tolerance) of q [nh, nt, dh] over the batch's pages, both [nh, nt, dh] doubles; rows of nobody (and of `skip`): NaN.

    Tolerance, from the kernel's roundings: o and each probability round once to the type (half a step, A = sum p |v| carries the
    latter); a probability below the type's normal numbers rounds to within LEAST, keys of them, over a row sum of at least 1; a
    score is a sum of dh products in f32, off by at most dh 2^-23 of sum |q k| (the matrix unit may cut instead of round), which
    moves p by that much relatively, above and below the fraction bar; ex2 and the sums add 2^-20 at most."""
    nh, dt = q.shape[0], q.dtype
    o = torch.full(q.shape, math.nan, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(o)
    for i, (n, l) in enumerate(zip(b.n, b.kv)):
        if n == 0 or i in skip:
            continue
        r0 = int(b.start[i])
        page, slot = b.slots(i, 0, l)
        for h in range(nh):
            kv = h // (nh // b.nkvh)
            k, v = b.k_pages[page, kv, slot].double(), b.v_pages[page, kv, slot].double()
            x = q[h, r0: r0 + n].double()
            s = x @ k.T * scale
            size = (x.abs() @ k.abs().T * abs(scale)).amax(-1, keepdim=True) if l else torch.zeros(n, 1, dtype=torch.float64, device=q.device)
            if causal:
                s = s.masked_fill(torch.arange(l, device=q.device)[None] > torch.arange(l - n, l, device=q.device)[:, None], -math.inf)
            m = s.amax(-1, keepdim=True) if l else torch.full((n, 1), -math.inf, dtype=torch.float64, device=q.device)
            p = torch.where(m == -math.inf, 0.0, torch.exp(s - torch.where(m == -math.inf, 0.0, m)))
            p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
            o[h, r0: r0 + n] = p @ v
            A = p @ v.abs()
            move = HALF_STEP[dt] + 2 * b.dh * 2.0 ** -23 * size + 2.0 ** -20
            vmax = v.abs().amax() if l else 0.0
            tol[h, r0: r0 + n] = HALF_STEP[dt] * o[h, r0: r0 + n].abs() + (1 + HALF_STEP[dt]) * (move * A + l * LEAST[dt] * vmax) + LEAST[dt]
    return o, tol
