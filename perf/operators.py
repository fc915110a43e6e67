"""Workloads of the operators of a paged serving batch: rope_norm, kv_append_paged and attention_paged.

A serving step holds `nt` rows of new tokens, packed sequence after sequence; sequence i owns rows
[seq_start[i], seq_start[i+1]) and its keys and values, the new ones included, lie in kv_len[i] cache slots that a page table maps.
`run` goes through one operator once: in plain torch operations, or (own = True) through the package's public calls.
"""
import functools
import importlib
import math
import random

import torch

own = False  # True: run() calls the package's operators; False: the plain form

LAYER = {"nh": 32, "nkvh": 8, "dh": 128}   # heads of the benchmark's layer
SHARD = {"nh": 4, "nkvh": 1, "dh": 128}    # the same layer cut over 8 ranks
THETA, EPS = 5e5, 1e-5


def listed():
    return [
        # one request writes its next token: the smallest call, latency only
        dict(LAYER, name="attn_one_token", op="attention", dtype="f16", nseq=1, chunks=0, new=1, past=1000, pad=0, ps=16, causal=True, lens=1),
        # a decode step of a busy server: ragged lengths, a captured batch with three rows unused
        dict(LAYER, name="attn_decode_61", op="attention", dtype="bf16", nseq=61, chunks=0, new=1, past=4095, pad=3, ps=16, causal=True, lens=2),
        # a decode step over long documents
        dict(LAYER, name="attn_decode_long", op="attention", dtype="f16", nseq=8, chunks=0, new=1, past=32100, pad=0, ps=64, causal=True, lens=3),
        # chunked prefill beside running requests: one chunk of a prompt, 31 single tokens
        dict(LAYER, name="attn_mixed", op="attention", dtype="bf16", nseq=32, chunks=1, new=487, past=2900, pad=0, ps=32, causal=True, lens=4),
        # a whole prompt of the benchmark's layer
        dict(LAYER, name="attn_prompt_4096", op="attention", dtype="f16", nseq=1, chunks=1, new=4096, past=0, pad=0, ps=16, causal=True, lens=5),
        # a later chunk of a long prompt on one rank of eight: few heads, many keys
        dict(SHARD, name="attn_chunk_shard", op="attention", dtype="bf16", nseq=1, chunks=1, new=1024, past=7001, pad=0, ps=64, causal=True, lens=6),
        # short documents that see all of themselves (scoring, embedding), small heads without sharing
        dict(name="attn_dense_dh64", op="attention", dtype="bf16", nseq=12, chunks=12, new=413, past=0, pad=0, ps=16, causal=False, lens=7, nh=16, nkvh=16, dh=64),
        # the step in front of it: a decode batch, plain rotation
        dict(LAYER, name="append_decode_61", op="append", dtype="f16", nseq=61, chunks=0, new=1, past=4095, pad=3, ps=16, norm=False, lens=2),
        # several prompts at once, with head norms
        dict(LAYER, name="append_prompts", op="append", dtype="bf16", nseq=9, chunks=7, new=1333, past=700, pad=5, ps=32, norm=True, lens=8),
        # queries and keys of a decode batch normed and rotated in the fused projection's output
        dict(LAYER, name="rope_norm_64", op="rope_norm", dtype="f16", nt=64, far=30000),
        # a ragged number of rows on a shard
        dict(SHARD, name="rope_norm_shard", op="rope_norm", dtype="bf16", nt=1777, far=9000),
        # a large prompt batch
        dict(LAYER, name="rope_norm_8192", op="rope_norm", dtype="bf16", nt=8192, far=130000),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    dtype = rng.choice(["f16", "bf16"])
    nh, nkvh, dh = rng.choice([(32, 8, 128), (4, 1, 128), (8, 2, 128), (16, 16, 64), (14, 2, 64), (12, 4, 96), (8, 1, 80), (5, 5, 128)])
    heads = {"nh": nh, "nkvh": nkvh, "dh": dh}
    op = rng.choice(["attention", "attention", "attention", "append", "rope_norm"])
    if op == "rope_norm":
        return dict(heads, op=op, dtype=dtype, nt=_spread(rng, 1, 8192), far=_spread(rng, 16, 200000))
    while True:
        kind = rng.choice(["decode", "mixed", "chunks"])
        nseq = _spread(rng, 1, 64 if kind == "decode" else 24)
        chunks = {"decode": 0, "mixed": (nseq + 3) // 4, "chunks": nseq}[kind]
        new = 1 if kind == "decode" else _spread(rng, 2, 4096)
        past = _spread(rng, 1, 33000) - 1
        case = dict(heads, op=op, dtype=dtype, nseq=nseq, chunks=chunks, new=new, past=past, pad=rng.choice([0, 0, 7]), ps=rng.choice([8, 16, 32, 64, 128]),
                    lens=rng.randrange(1 << 20))
        if op == "append":
            case["norm"] = rng.random() < 0.5
            if sum(_lengths(case)[0]) <= 8192:
                return case
        else:
            case["causal"] = rng.random() < 0.8
            w = work(case)
            n, kv = _lengths(case)
            # no more than the largest listed case, and a plain form that fits (scores and keys are padded to the longest)
            if w["flops"] <= 1.3e11 and w["bytes"] <= 1.0e9 and nseq * max(kv) * max(max(n) * nh, 2 * nkvh * dh) <= 0.5e9:
                return case


def _lengths(case):
    """New tokens and cache slots of every sequence: fixed by the case (the first sequence has the longest past and chunk)."""
    r = random.Random(case["lens"])
    n = [1] * case["nseq"]
    for i in range(case["chunks"]):
        n[i] = case["new"] if i == 0 else r.randint(max(1, case["new"] // 3), case["new"])
    kv = [x + (case["past"] if i == 0 else r.randint(case["past"] // 8, case["past"])) for i, x in enumerate(n)]
    return n, kv


def _dtype(case):
    return {"f16": torch.float16, "bf16": torch.bfloat16}[case["dtype"]]


def work(case):
    nh, nkvh, dh = case["nh"], case["nkvh"], case["dh"]
    if case["op"] == "rope_norm":
        rows = case["nt"] * (nh + nkvh)
        return {"bytes": rows * dh * 4 + case["nt"] * 4 + (nh + nkvh) * dh * 2, "flops": rows * dh * 7}
    n, kv = _lengths(case)
    nt = sum(n)
    if case["op"] == "append":
        return {"bytes": nt * dh * 2 * (2 * nh + 4 * nkvh) + nt * 8, "flops": nt * dh * (nh + nkvh) * (7 if case["norm"] else 3)}
    seen = sum(x * (l - x) + x * (x + 1) // 2 if case["causal"] else x * l for x, l in zip(n, kv))
    return {"bytes": 4 * nt * nh * dh + 4 * sum(kv) * nkvh * dh + 4 * sum(-(-l // case["ps"]) for l in kv), "flops": 4 * nh * dh * seen}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt, nh, nkvh, dh = _dtype(case), case["nh"], case["nkvh"], case["dh"]

    def normal(*shape, std=1.0):
        return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, std, generator=g).to(dt)

    s = {"case": case}
    if case["op"] == "rope_norm":
        nt = case["nt"]
        s["qkv"] = normal(nt, (nh + 2 * nkvh) * dh)  # the fused projection's output; its q and k heads are the operand
        s["pos"] = torch.randint(0, case["far"], (nt,), generator=g, device="cuda").to(torch.int32)
        s["w"] = (1.0 + 0.2 * normal(nh + nkvh, dh).float()).to(dt)
        s["y"] = torch.zeros(nt, nh + nkvh, dh, dtype=dt, device="cuda")
        return s
    n, kv = _lengths(case)
    ps, nseq, nt = case["ps"], case["nseq"], sum(n) + case["pad"]
    pages = [-(-l // ps) for l in kv]
    npages = sum(pages) + 3
    order = torch.randperm(npages, generator=g, device="cuda").to(torch.int32)
    first = torch.tensor([sum(pages[:i]) for i in range(nseq)], device="cuda")
    count = torch.tensor(pages, device="cuda")
    col = torch.arange(max(pages), device="cuda")
    s["page_table"] = torch.where(col[None] < count[:, None], order[(first[:, None] + col[None]).clamp(max=npages - 1)], 0).to(torch.int32)
    s["seq_start"] = torch.tensor([sum(n[:i]) for i in range(nseq + 1)], dtype=torch.int32, device="cuda")
    s["kv_len"] = torch.tensor(kv, dtype=torch.int32, device="cuda")
    s["max_seq"] = max(n)
    s["qkv"] = normal(nt, (nh + 2 * nkvh) * dh)
    if case["op"] == "attention":
        # queries stretched so that a row's weights differ by orders of magnitude, as trained heads' do
        s["qkv"][:, : nh * dh] = (2.5 * s["qkv"][:, : nh * dh].float()).to(dt)
        s["k_pages"], s["v_pages"] = normal(npages, nkvh, ps, dh), normal(npages, nkvh, ps, dh)
        s["o"] = torch.zeros(nt, nh, dh, dtype=dt, device="cuda")
    else:
        s["k_pages"], s["v_pages"] = (torch.zeros(npages, nkvh, ps, dh, dtype=dt, device="cuda") for _ in range(2))
        at = torch.tensor([l - x for x, l in zip(n, kv)], device="cuda")
        seq = torch.repeat_interleave(torch.arange(nseq, device="cuda"), torch.tensor(n, device="cuda"))
        pos = torch.arange(sum(n), device="cuda") - s["seq_start"][seq] + at[seq]
        s["pos"] = torch.cat([pos, torch.zeros(case["pad"], dtype=pos.dtype, device="cuda")]).to(torch.int32)
        s["w"] = (1.0 + 0.2 * normal(nh + nkvh, dh).float()).to(dt) if case["norm"] else None
        s["q_out"] = torch.zeros(nt, nh, dh, dtype=dt, device="cuda")
    return s


def _heads(s):
    """Views of the fused projection's output: q, k and v heads, [rows, heads, dh]."""
    c = s["case"]
    t = s["qkv"].view(s["qkv"].shape[0], c["nh"] + 2 * c["nkvh"], c["dh"])
    return t[:, : c["nh"]], t[:, c["nh"]: c["nh"] + c["nkvh"]], t[:, c["nh"] + c["nkvh"]:]


def _norm_rotate(x, pos, w):
    """[rows, heads, dh] in 32 bits (angles in 64): optional norm of every head, rotation of adjacent pairs."""
    dh = x.shape[-1]
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    angle = pos.double()[:, None] * THETA ** (-torch.arange(0, dh, 2, dtype=torch.float64, device=x.device) / dh)[None]
    c, n = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * n, a * n + b * c], -1).flatten(-2)


def _plain_attention(s):
    c, q = s["case"], _heads(s)[0]
    nh, nkvh, dh, ps = c["nh"], c["nkvh"], c["dh"], c["ps"]
    group, nseq, most = nh // nkvh, c["nseq"], s["max_seq"]
    start, kv = s["seq_start"].long(), s["kv_len"].long()
    n = start[1:] - start[:-1]
    j = torch.arange(most, device="cuda")
    live = j[None] < n[:, None]
    row = torch.where(live, start[:-1, None] + j[None], 0)
    qs = q[row].float().view(nseq, most, nkvh, group, dh).permute(0, 2, 3, 1, 4).reshape(nseq, nkvh, group * most, dh)
    table = s["page_table"].long()
    k = s["k_pages"][table].permute(0, 2, 1, 3, 4).reshape(nseq, nkvh, -1, dh).float()
    v = s["v_pages"][table].permute(0, 2, 1, 3, 4).reshape(nseq, nkvh, -1, dh).float()
    at = torch.arange(k.shape[2], device="cuda")
    v = torch.where((at[None] < kv[:, None])[:, None, :, None], v, 0.0)
    last = (kv - n)[:, None] + j[None] if c["causal"] else (kv - 1)[:, None].expand(-1, most)
    seen = at[None, None] <= last[..., None]  # [nseq, most, keys]
    x = (qs @ k.transpose(-1, -2)).view(nseq, nkvh, group, most, -1) * dh ** -0.5
    x = torch.where(seen[:, None, None], x, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-3e38))
    total = x.sum(-1, keepdim=True)
    y = (x.view(nseq, nkvh, group * most, -1) @ v).view(nseq, nkvh, group, most, dh) / torch.where(total > 0, total, 1.0)
    y = y.permute(0, 3, 1, 2, 4).reshape(nseq, most, nh, dh).to(q.dtype)
    o = torch.zeros(q.shape[0] + 1, nh, dh, dtype=q.dtype, device="cuda")
    o[torch.where(live, row, q.shape[0])] = y  # what stands for no token goes to the row behind the last
    return o[:-1]


def _plain_append(s):
    c = s["case"]
    q, k, v = _heads(s)
    nh, ps = c["nh"], c["ps"]
    start, kv = s["seq_start"].long(), s["kv_len"].long()
    rows = torch.arange(q.shape[0] - c["pad"], device="cuda")
    seq = torch.searchsorted(start, rows, right=True) - 1
    slot = kv[seq] - start[seq + 1] + rows
    page, at = s["page_table"].long()[seq, slot // ps], slot % ps
    live, w = rows.shape[0], s["w"]
    q_out = torch.zeros_like(s["q_out"])
    q_out[:live] = _norm_rotate(q[:live], s["pos"][:live], None if w is None else w[:nh]).to(q.dtype)
    s["k_pages"][page, :, at] = _norm_rotate(k[:live], s["pos"][:live], None if w is None else w[nh:]).to(k.dtype)
    s["v_pages"][page, :, at] = v[:live]
    return {"q": q_out, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


@functools.lru_cache(maxsize=None)
def _operators():
    """The handles that a program makes once."""
    ops = importlib.import_module("operators-rs_b200")
    return ops, ops.Rope(0), ops.KvAppendPaged(0), ops.AttentionPaged(0)


def _own(s):
    ops, rope, append, attention = _operators()
    c = s["case"]
    q, k, v = _heads(s)
    if c["op"] == "rope_norm":
        qk = s["qkv"].view(c["nt"], -1, c["dh"])[:, : c["nh"] + c["nkvh"]]
        rope.launch_norm(ops.RopeNormArgs.of(s["y"], qk, s["pos"].view(torch.uint32), s["w"], EPS, THETA))
        return s["y"]
    batch = ops.PagedBatch(s["page_table"], s["seq_start"], s["kv_len"], s["max_seq"])
    if c["op"] == "append":
        append.launch(ops.KvAppendPagedArgs.of(s["q_out"], q, k, v, s["k_pages"], s["v_pages"], s["pos"].view(torch.uint32), batch, THETA, s["w"], EPS))
        return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    args = ops.AttentionPagedArgs.of(q.permute(1, 0, 2), s["k_pages"], s["v_pages"], s["o"].permute(1, 0, 2), batch,
                                     ops.MASK_CAUSAL if c["causal"] else ops.MASK_NONE)
    if "workspace" not in s:  # scratch that a program keeps beside its buffers
        s["workspace"] = torch.empty(attention.scheme(args), dtype=torch.uint8, device="cuda")
    attention.launch(args, s["workspace"])
    return s["o"]


def run(s):
    if own:
        return _own(s)
    if s["case"]["op"] == "rope_norm":
        qk = s["qkv"].view(s["case"]["nt"], -1, s["case"]["dh"])[:, : s["y"].shape[1]]
        return _norm_rotate(qk, s["pos"], s["w"]).to(s["y"].dtype)
    return _plain_append(s) if s["case"]["op"] == "append" else _plain_attention(s)


def exact(case, seed):
    """The operators' definitions in 64 bits, sequence by sequence and head by head."""
    s = prepare(case, seed)
    nh, nkvh, dh = case["nh"], case["nkvh"], case["dh"]
    t = s["qkv"].double().view(-1, nh + 2 * nkvh, dh)

    def turned(x, pos, w):
        if w is not None:
            x = x / ((x ** 2).sum(-1, keepdim=True) / dh + EPS).sqrt() * w.double()
        z = torch.view_as_complex(x.reshape(*x.shape[:-1], dh // 2, 2).contiguous())
        turn = pos.double()[:, None, None] * torch.exp(-math.log(THETA) * 2 * torch.arange(dh // 2, device="cuda").double() / dh)
        return torch.view_as_real(z * torch.polar(torch.ones_like(turn), turn)).flatten(-2)

    if case["op"] == "rope_norm":
        return turned(t[:, : nh + nkvh], s["pos"], s["w"])
    start, kv, ps = s["seq_start"].tolist(), s["kv_len"].tolist(), case["ps"]
    if case["op"] == "append":
        out = {"q": s["q_out"].double(), "k_pages": s["k_pages"].double(), "v_pages": s["v_pages"].double()}
        for i in range(case["nseq"]):
            b, e = start[i], start[i + 1]
            heads = turned(t[b:e, : nh + nkvh], s["pos"][b:e], s["w"])
            at = torch.arange(kv[i] - (e - b), kv[i], device="cuda")
            page = s["page_table"][i].long()[at // ps]
            out["q"][b:e] = heads[:, :nh]
            out["k_pages"][page, :, at % ps] = heads[:, nh:]
            out["v_pages"][page, :, at % ps] = t[b:e, nh + nkvh:]
        return out
    o = s["o"].double()
    for i in range(case["nseq"]):
        b, e, l = start[i], start[i + 1], kv[i]
        page = s["page_table"][i, : -(-l // ps)].long()
        hidden = None
        if case["causal"]:
            hidden = torch.arange(l, device="cuda")[None] > torch.arange(l - (e - b), l, device="cuda")[:, None]
        for h in range(nkvh):
            k = s["k_pages"][page, h].reshape(-1, dh)[:l].double()
            v = s["v_pages"][page, h].reshape(-1, dh)[:l].double()
            for f in range(h * (nh // nkvh), (h + 1) * (nh // nkvh)):
                x = t[b:e, f] @ k.T / math.sqrt(dh)
                if hidden is not None:
                    x.masked_fill_(hidden, -math.inf)
                o[b:e, f] = torch.softmax(x, -1) @ v
    return o
