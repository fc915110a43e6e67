"""The operators of a paged serving batch (rope_norm, kv_append_paged, attention_paged) against plain 64-bit forms
(paged_reference.py, which also derives the tolerances): head layouts, page sizes that end inside a tile, cache layouts, lengths
from nothing to long ones, rows of nobody, what lies in unused slots, bad pages and lengths, graphs, and a step made of them."""
import importlib
import math

import pytest
import torch

import __graft_entry__ as graft
import paged_reference as ref

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
THETA, EPS = 5e5, 1e-5


@pytest.fixture(scope="module")
def ops(pkg, dev):
    class Ops:
        rope, append, attention = pkg.Rope(0), pkg.KvAppendPaged(0), pkg.AttentionPaged(0)
    return Ops


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def normal(g, shape, dt, std=1.0):
    return (std * torch.randn(shape, generator=g, device=g.device)).to(dt)


def near(got, want, tol, what):
    """Where `want` is NaN (rows of nobody) nothing is compared here."""
    there = ~torch.isnan(want)
    d = (got.double() - want).abs()
    bad = there & ~(d <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {int(there.sum())} off, first at {bad.nonzero()[0].tolist()}: got {got[bad][0].item()}, " \
                          f"want {want[bad][0].item()} within {tol[bad][0].item()}"


# ------------------------------------------------------------------------------------------------ rope_norm
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("nt,nh,dh,far", [(1, 1, 8, 1), (1, 40, 128, 1), (3, 5, 64, 100), (7, 6, 80, 5000), (33, 16, 96, 9000), (129, 10, 256, 40), (700, 40, 128, 200000),
                                          (5000, 5, 128, 4000000000)])
def test_rope_norm(pkg, dev, ops, dt, nt, nh, dh, far):
    g = gen(dev, nt)
    buf = normal(g, (nt, nh + 3, dh), dt, 3.0)
    x = buf[:, 1: nh + 1]
    pos = torch.randint(0, far, (nt,), generator=g, device=dev)
    w = (1 + 0.3 * torch.randn(nh, dh, generator=g, device=dev)).to(dt)
    y = torch.empty(nt, nh, dh, dtype=dt, device=dev)
    ops.rope.launch_norm(pkg.RopeNormArgs.of(y, x, pos.to(torch.uint32), w, EPS, THETA))
    want = ref.rotate(x.double(), pos, THETA, w, EPS)
    near(y, want, ref.rotate_tolerance(x.double(), pos, THETA, w, EPS, dt, want), "rope_norm")
    # in place, one weight row of f32 for all heads, 64-bit positions; the heads beside stay as they are
    before = buf.clone()
    w32 = 1 + 0.3 * torch.randn(1, dh, generator=g, device=dev)
    want = ref.rotate(x.double(), pos, 1e4, w32, 0.5)
    tol = ref.rotate_tolerance(x.double(), pos, 1e4, w32, 0.5, dt, want)
    ops.rope.launch_norm(pkg.RopeNormArgs(x, x, x, x, pkg.TensorLayout.new_contiguous(pkg.U64, (nt,)), pos, w32.expand(nh, dh), w32, 0.5, 1e4))
    near(x, want, tol, "rope_norm in place")
    assert torch.equal(buf[:, :1], before[:, :1]) and torch.equal(buf[:, nh + 1:], before[:, nh + 1:])


def test_rope_norm_of_zeros_and_strides(pkg, dev, ops):
    """A head of zeros stays zeros (epsilon keeps the root away from 0); heads in front of tokens in memory; positions with a stride."""
    g = gen(dev, 5)
    x = normal(g, (6, 9, 64), F16).transpose(0, 1)  # [9 tokens, 6 heads, 64], heads outermost in memory
    x[2, 3] = 0
    pos = torch.arange(0, 36, device=dev, dtype=torch.int32)[::4]
    y = torch.empty(9, 6, 64, dtype=F16, device=dev)
    w = torch.ones(6, 64, dtype=F16, device=dev)
    ops.rope.launch_norm(pkg.RopeNormArgs(y, y, x, x, pkg.TensorLayout(pkg.U32, (9,), (16,)), pos, w, w, EPS, THETA))
    want = ref.rotate(x.double(), pos, THETA, w, EPS)
    near(y, want, ref.rotate_tolerance(x.double(), pos, THETA, w, EPS, F16, want), "rope_norm strides")
    assert not y[2, 3].any()


# ------------------------------------------------------------------------------------------------ kv_append_paged
APPEND = [  # n, kv, heads, dh, page, order, pad
    ([1], [1], (1, 1), 8, 8, "page_head_slot", 0),
    ([1] * 61, [1 + 37 * i % 300 for i in range(61)], (32, 8), 128, 16, "page_head_slot", 3),
    ([5, 0, 130, 1, 17], [5, 9, 200, 64, 33], (8, 2), 64, 32, "page_slot_head", 0),
    ([70, 33], [1000, 33], (6, 3), 96, 128, "joint", 9),
    ([0, 3, 0, 0, 4, 0], [0, 3, 0, 7, 4, 0], (4, 4), 256, 8, "page_head_slot", 1),
]


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("case", range(len(APPEND)))
def test_kv_append_paged(pkg, dev, ops, dt, norm, case):
    n, kv, (nh, nkvh), dh, ps, order, pad = APPEND[case]
    b = ref.Batch(dev, dt, n, kv, nkvh, dh, ps, pad=pad, seed=case, order=order, first=2 if pad else 0)
    g = gen(dev, case)
    qkv = normal(g, (b.nt, nh + 2 * nkvh, dh), dt)
    q, k, v = qkv[:, :nh], qkv[:, nh: nh + nkvh], qkv[:, nh + nkvh:]
    w = (1 + 0.3 * torch.randn(nh + nkvh, dh, generator=g, device=dev)).to(dt) if norm else None
    live = slice(b.first, b.first + sum(n))
    pos = torch.zeros(b.nt, dtype=torch.int64)
    pos[live] = torch.cat([torch.arange(l - m, l) for m, l in zip(n, kv)])
    pos = pos.to(dev)
    want = ref.rotate(qkv[:, : nh + nkvh].double(), pos, THETA, w, EPS)
    tol = ref.rotate_tolerance(qkv[:, : nh + nkvh].double(), pos, THETA, w, EPS, dt, want)
    q_out = torch.full((b.nt, nh, dh), 7.0, dtype=dt, device=dev)
    k_want, v_want = b.k_pages.double(), b.v_pages.double()
    k_tol = torch.zeros_like(k_want)
    for i, (m, l) in enumerate(zip(n, kv)):
        if m:
            r = int(b.start[i])
            page, slot = b.slots(i, l - m, l)
            k_want[page, :, slot], v_want[page, :, slot] = want[r: r + m, nh:], v[r: r + m].double()
            k_tol[page, :, slot] = tol[r: r + m, nh:]
    ops.append.launch(pkg.KvAppendPagedArgs.of(q_out, q, k, v, b.k_pages, b.v_pages, pos.to(torch.uint32), b.descriptor(pkg), THETA, w, EPS))
    assert ops.append.status() == 0
    near(q_out[live], want[live, :nh], tol[live, :nh], "q")
    near(b.k_pages, k_want, k_tol, "keys")
    assert torch.equal(torch.isnan(b.k_pages), torch.isnan(k_want)) and torch.equal(torch.isnan(b.v_pages), torch.isnan(v_want))  # nothing else written
    assert torch.equal(torch.nan_to_num(b.v_pages), torch.nan_to_num(v_want).to(dt))
    q_out[live] = 7.0
    assert bool((q_out == 7.0).all())  # rows of nobody
    # in place
    ops.append.launch(pkg.KvAppendPagedArgs.of(q, q, k, v, b.k_pages, b.v_pages, pos.to(torch.uint32), b.descriptor(pkg), THETA, w, EPS))
    near(q[live], want[live, :nh], tol[live, :nh], "q in place")


def test_kv_append_paged_reports_and_survives_bad_batches(pkg, dev, ops):
    op = pkg.KvAppendPaged(0)

    def step(bend):
        b = ref.Batch(dev, F16, [3, 2], [20, 9], 2, 64, 8, seed=3)
        qkv = normal(gen(dev, 1), (b.nt, 8, 64), F16)
        bend(b)
        pos = torch.arange(5, dtype=torch.int32, device=dev).view(torch.uint32)
        op.launch(pkg.KvAppendPagedArgs.of(qkv[:, :4].clone(), qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], b.k_pages, b.v_pages, pos, b.descriptor(pkg), THETA))
        code = op.status()
        op.status_reset()
        return b, code, int((~torch.isnan(b.v_pages)).sum()) // 128

    def page(b):
        b.page_table[0, 2] = b.npages
    b, code, written = step(page)  # tokens 17..19 of sequence 0: slots 17, 18, 19 lie in its page 2
    assert (code, written) == (pkg.PAGED_BAD_PAGE, 2)

    def minus(b):
        b.page_table[0, 2] = -1
    assert step(minus)[1:] == (pkg.PAGED_BAD_PAGE, 2)

    def short(b):
        b.kv_len[0] = 1  # three new tokens, one slot: the last one gets it
    assert step(short)[1:] == (pkg.PAGED_BAD_LENGTH, 3)

    def long(b):
        b.kv_len[0] = 33  # the table is 4 wide (one entry behind the last page): 32 slots, its fourth page is nobody's
        b.page_table[0, 3] = b.page_table[0, 2]
    b, code, written = step(long)
    assert code == pkg.PAGED_BAD_LENGTH and written == 4  # slots 30, 31 and sequence 1's two

    def negative(b):
        b.kv_len[0] = -5
    assert step(negative)[1:] == (pkg.PAGED_BAD_LENGTH, 2)

    def rows(b):
        b.seq_start[1] = 900  # sequence 0 cut to the step's rows, sequence 1 starts behind them
    b, code, written = step(rows)
    assert code in (pkg.PAGED_BAD_ROWS, pkg.PAGED_BAD_LENGTH)
    assert step(lambda b: None)[1:] == (0, 5)


# ------------------------------------------------------------------------------------------------ attention_paged
def attend(pkg, op, b, q, o, causal=True, scale=None, ws=None):
    args = pkg.AttentionPagedArgs.of(q, b.k_pages, b.v_pages, o, b.descriptor(pkg), pkg.MASK_CAUSAL if causal else pkg.MASK_NONE, scale)
    if ws is None:
        ws = torch.full((op.scheme(args),), 0xff, dtype=torch.uint8, device=q.device)  # NaN patterns: nothing may be read before it is written
    op.launch(args, ws)
    return ws


def check_attention(pkg, dev, op, b, nh, causal=True, scale=None, std=2.0, skip=(), status=0):
    g = gen(dev, sum(b.kv) + nh)
    b.fill(g)
    qkv = normal(g, (b.nt, nh + 2, b.dh), b.dt, std)
    q = qkv[:, 1: nh + 1].permute(1, 0, 2)
    o = torch.full((b.nt, nh + 1, b.dh), 7.0, dtype=b.dt, device=dev)[:, :nh].permute(1, 0, 2)
    attend(pkg, op, b, q, o, causal, scale)
    assert op.status() == status
    want, tol = ref.attention(b, q, causal, b.dh ** -0.5 if scale is None else scale, skip)
    near(o, want, tol, "o")
    assert bool((o[torch.isnan(want)] == 7.0).all()), "rows of nobody were written"


ATTENTION = [  # n, kv, (nh, nkvh), dh, page, order, pad
    ([1], [1], (1, 1), 8, 8, "page_head_slot", 0),
    ([1], [777], (32, 8), 128, 16, "page_head_slot", 0),
    ([1] * 9, [1, 2, 15, 16, 17, 127, 128, 129, 300], (8, 2), 128, 16, "page_head_slot", 0),
    ([1] * 5, [4, 0, 250, 0, 33], (4, 4), 64, 8, "page_slot_head", 4),                   # sequences without a single slot
    ([1] * 3, [500, 40, 3000], (16, 1), 128, 32, "joint", 0),
    ([1] * 4, [130, 129, 128, 1], (12, 4), 96, 64, "page_head_slot", 0),
    ([1] * 2, [90, 700], (8, 1), 80, 128, "page_slot_head", 2),
    ([4, 3, 2], [300, 3, 129], (8, 2), 128, 16, "page_head_slot", 0),                    # a few drafted tokens each
    ([2, 1, 2], [60, 17, 900], (32, 4), 64, 256, "page_head_slot", 0),
    ([17], [17], (8, 2), 128, 16, "page_head_slot", 0),
    ([33, 0, 1, 65, 1], [33, 12, 500, 190, 1], (8, 2), 128, 16, "page_head_slot", 5),    # chunks beside single tokens and an idle sequence
    ([128], [128], (4, 4), 64, 64, "page_slot_head", 0),
    ([129, 127], [400, 127], (2, 2), 128, 128, "joint", 0),
    ([300], [1500], (14, 2), 64, 16, "page_head_slot", 1),                               # 7 query heads per kv head
    ([257, 40], [257, 1000], (5, 5), 128, 8, "page_head_slot", 0),
    ([100], [333], (12, 4), 96, 32, "page_slot_head", 0),
    ([70, 9], [70, 520], (8, 1), 80, 16, "page_head_slot", 0),
    ([50], [300], (40, 1), 24, 16, "page_head_slot", 0),
    ([20, 1], [7, 0], (8, 2), 128, 16, "page_head_slot", 0),                             # more new tokens than slots: rows that see nothing
    ([600], [3], (4, 1), 64, 16, "page_head_slot", 0),
    ([3], [200], (128, 1), 64, 16, "page_head_slot", 0),
    ([513], [4100], (2, 1), 128, 1024, "page_head_slot", 0),
]


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", range(len(ATTENTION)))
def test_attention_paged(pkg, dev, ops, dt, causal, case):
    n, kv, (nh, nkvh), dh, ps, order, pad = ATTENTION[case]
    # max_seq: known, unknown
    b = ref.Batch(dev, dt, n, kv, nkvh, dh, ps, pad=pad, seed=case, order=order, first=pad // 2, max_seq=max(n) if case % 3 else 0,
                  index=torch.uint32 if case % 2 else torch.int32)
    check_attention(pkg, dev, ops.attention, b, nh, causal)


def test_attention_paged_many_sequences(pkg, dev, ops):
    """More sequences than threads of a block, lengths from 0 to 200, a few chunks between them."""
    n = [1 if i % 50 else 40 for i in range(1500)]
    kv = [n[i] + (i * 37) % 160 if i % 11 else (0 if n[i] == 1 else 40) for i in range(1500)]
    check_attention(pkg, dev, ops.attention, ref.Batch(dev, F16, n, kv, 1, 64, 16, seed=1), 2)


@pytest.mark.parametrize("nseq,nh,nkvh,dh,new,most", [(700, 16, 1, 128, 1, 120), (400, 6, 2, 80, 2, 200), (500, 8, 8, 64, 1, 90), (450, 14, 2, 64, 2, 330)])
def test_attention_paged_many_short_sequences(pkg, dev, ops, nseq, nh, nkvh, dh, new, most):
    """Sequences that one warp takes alone, some of nothing, some too long for that, the last ones of a share taken together."""
    kv = [(i * 53) % most + new if i % 17 else (0 if i % 2 else 5 * most) for i in range(nseq)]
    check_attention(pkg, dev, ops.attention, ref.Batch(dev, BF16 if nseq % 2 else F16, [new] * nseq, kv, nkvh, dh, 16, seed=2, max_seq=new), nh)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n,kv,nh,nkvh,dh", [([1] * 20 + [200], [3000 + 7 * i for i in range(20)] + [900], 8, 2, 128),       # long single tokens: side by side
                                             ([1, 600, 1, 500], [300, 700, 40, 500], 4, 2, 64),                              # a small share of the work
                                             ([1] * 60 + [90, 1], [60 + i for i in range(60)] + [4000, 9], 16, 2, 64),       # short ones beside a long past
                                             ([2] * 40 + [300], [1500] * 40 + [1300], 4, 4, 96)])
def test_attention_paged_chunks_beside_single_tokens(pkg, dev, ops, causal, n, kv, nh, nkvh, dh):
    check_attention(pkg, dev, ops.attention, ref.Batch(dev, BF16, n, kv, nkvh, dh, 32, seed=4, pad=2), nh, causal)


@pytest.mark.parametrize("n,kv", [([1], [40000]), ([1, 1], [30, 20001]), ([200], [20000]), ([2, 64], [16000, 9001])])
def test_attention_paged_long(pkg, dev, ops, n, kv):
    check_attention(pkg, dev, ops.attention, ref.Batch(dev, BF16, n, kv, 2, 128, 64, seed=9), 8)


@pytest.mark.parametrize("n,kv", [([1, 1], [300, 5]), ([150], [400])])
def test_attention_paged_scale_and_large_scores(pkg, dev, ops, n, kv):
    """Scores of several hundred and a scale of the caller's: the running maximum carries them."""
    check_attention(pkg, dev, ops.attention, ref.Batch(dev, F16, n, kv, 2, 64, 16, seed=2), 4, scale=1.0, std=6.0)
    check_attention(pkg, dev, ops.attention, ref.Batch(dev, F16, n, kv, 2, 64, 16, seed=2), 4, scale=-0.25)
    check_attention(pkg, dev, ops.attention, ref.Batch(dev, F16, n, kv, 2, 64, 16, seed=2), 4, scale=0.0)


def test_attention_paged_masked_infinities(pkg, dev, ops):
    """A later token's key of infinities and value of NaN show in no earlier row of another tile or sequence; scores of minus
    infinity (a key of -inf against positive queries) weigh nothing."""
    b = ref.Batch(dev, F16, [1, 1], [200, 64], 1, 64, 16, seed=4)
    g = gen(dev, 4)
    b.fill(g)
    page, slot = b.slots(0, 50, 51)
    b.k_pages[page, :, slot] = -math.inf
    q = normal(g, (2, 2, 64), F16).abs() + 0.1
    o = torch.zeros_like(q)
    attend(pkg, ops.attention, b, q, o)
    b.k_pages[page, :, slot] = -60000.0  # its weight is 2^-huge: the oracle without an infinity times zero
    want, tol = ref.attention(b, q, True, 0.125)
    tol = tol.clamp(max=0.02)
    near(o, want, tol, "o")


def test_attention_paged_reports_and_survives_bad_batches(pkg, dev):
    op = pkg.AttentionPaged(0)

    def step(n, kv, bend, max_seq=0):
        b = ref.Batch(dev, F16, n, kv, 2, 64, 16, seed=3, max_seq=max_seq)
        g = gen(dev, 1)
        b.fill(g)
        q = normal(g, (4, b.nt, 64), F16)
        want, tol = ref.attention(b, q, True, 0.125)
        bend(b)
        o = torch.full_like(q, 7.0)
        attend(pkg, op, b, q, o)
        code = op.status()
        op.status_reset()
        assert op.status() == 0
        return b, q, o, want, tol, code

    for n, kv in (([1, 1], [100, 40]), ([40, 50], [100, 90])):
        # a page outside: its slots read as zeros, the other sequence is untouched
        def page(b):
            b.page_table[0, 2] = b.npages
        b, q, o, want, tol, code = step(n, kv, page)
        assert code == pkg.PAGED_BAD_PAGE
        near(o[:, n[0]:], want[:, n[0]:], tol[:, n[0]:], "the other sequence")
        b.table[0, 2] = b.spares[0]  # a page of nobody, as zeros
        b.k_pages[b.spares[0]] = 0
        b.v_pages[b.spares[0]] = 0
        near(o, *ref.attention(b, q, True, 0.125), "zeros for the missing page")

        # more slots than the table can map: cut
        def long(b):
            b.kv_len[1] = 100000
            b.page_table[1, -(-kv[1] // 16):] = b.spares[0]
            b.v_pages[b.spares[0]] = 0
            b.k_pages[b.spares[0]] = 0
        b, q, o, want, tol, code = step(n, kv, long)
        assert code == pkg.PAGED_BAD_LENGTH and bool(torch.isfinite(o[:, : n[0]]).all())
        near(o[:, : n[0]], want[:, : n[0]], tol[:, : n[0]], "the other sequence")

        # rows: sequence 1 claims rows behind the step's, and one that starts before the one in front of it
        def rows(b):
            b.seq_start[2] = 5000
        b, q, o, want, tol, code = step(n, kv, rows)
        assert code == pkg.PAGED_BAD_ROWS
        near(o, want, tol, "cut to the step's rows")
        def falling(b):
            b.seq_start[2] = 0
        b, q, o, want, tol, code = step(n, kv, falling)
        assert code == pkg.PAGED_BAD_ROWS
        near(o[:, : n[0]], want[:, : n[0]], tol[:, : n[0]], "the first sequence")
        assert bool((o[:, n[0]:] == 7.0).all())
    # longer than promised: left as it is
    b, q, o, want, tol, code = step([1, 3, 1], [50, 60, 70], lambda b: None, max_seq=2)
    assert code == pkg.PAGED_BAD_ROWS and bool((o[:, 1:4] == 7.0).all())
    near(o[:, [0, 4]], want[:, [0, 4]], tol[:, [0, 4]], "the others")
    b, q, o, want, tol, code = step([1, 90, 40], [50, 160, 70], lambda b: None, max_seq=80)
    assert code == pkg.PAGED_BAD_ROWS and bool((o[:, 1:91] == 7.0).all())
    near(o[:, 91:], want[:, 91:], tol[:, 91:], "the others")


@pytest.mark.parametrize("n,kv,n2,kv2", [([1] * 6, [300, 2, 90, 1000, 17, 64], [1, 1, 1, 1, 0, 0], [310, 1, 1000, 20, 0, 5]),
                                         ([40, 1, 100], [700, 33, 100], [1, 1, 90], [5, 600, 600])])
def test_attention_paged_graph_replayed_with_other_lengths(pkg, dev, ops, n, kv, n2, kv2):
    """A captured launch reads the batch when it runs."""
    b = ref.Batch(dev, F16, [max(x, y) for x, y in zip(n, n2)], [max(x, y) for x, y in zip(kv, kv2)], 2, 128, 16, seed=6)
    g = gen(dev, 6)
    b.fill(g)
    q = normal(g, (8, b.nt, 128), F16)
    o = torch.full_like(q, 7.0)

    def use(n, kv):
        b.n, b.kv = n, kv
        b.start = torch.tensor([sum(n[:i]) for i in range(len(n) + 1)])
        b.seq_start.copy_(b.start)
        b.kv_len.copy_(torch.tensor(kv))

    use(n, kv)
    ws = attend(pkg, ops.attention, b, q, o)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attend(pkg, ops.attention, b, q, o, ws=ws)
    for lens in ((n2, kv2), (n, kv), (n2, kv2)):
        use(*lens)
        o.fill_(7.0)
        ws.fill_(0xff)
        graph.replay()
        want, tol = ref.attention(b, q, True, 128 ** -0.5)
        near(o, want, tol, "o")
        assert bool((o[torch.isnan(want)] == 7.0).all())
    assert ops.attention.status() == 0


def test_attention_paged_two_streams_at_once(pkg, dev, ops):
    """One handle, two streams, a workspace each."""
    made = []
    for k in range(2):
        b = ref.Batch(dev, BF16, [1] * 7 if k else [80, 1], [900 + 100 * i for i in range(7)] if k else [2000, 800], 2, 128, 16, seed=k)
        g = gen(dev, k)
        b.fill(g)
        q = normal(g, (8, b.nt, 128), BF16)
        made.append((b, q, torch.zeros_like(q), torch.cuda.Stream(dev)))
    torch.cuda.synchronize()
    for _ in range(20):
        for b, q, o, s in made:
            with torch.cuda.stream(s):
                attend(pkg, ops.attention, b, q, o)
    torch.cuda.synchronize()
    for b, q, o, s in made:
        near(o, *ref.attention(b, q, True, 128 ** -0.5), "o")


def test_attention_paged_repeats_bit_for_bit(pkg, dev, ops):
    b = ref.Batch(dev, F16, [1, 1, 60, 1], [5000, 80, 3000, 64], 2, 128, 16, seed=8)
    g = gen(dev, 8)
    b.fill(g)
    q = normal(g, (8, b.nt, 128), F16)
    outs = []
    for _ in range(3):
        o = torch.zeros_like(q)
        attend(pkg, ops.attention, b, q, o)
        outs.append(o)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("n,kv,nkvh,nh", [([1], [9000], 9, 18), ([1, 1, 1], [12000, 11000, 12500], 3, 3), ([40], [12000], 9, 36), ([20, 30, 300], [9000, 9500, 9800], 3, 12)])
def test_attention_paged_units_of_many_parts(pkg, dev, ops, n, kv, nkvh, nh):
    """Nine units over all SMs: 17 or 18 parts each, joined in two rounds; the second unit's first part is the CTA of the first
    unit's last one.  Over and over: nothing depends on who comes when."""
    b = ref.Batch(dev, F16, n, kv, nkvh, 128, 16, seed=5)
    g = gen(dev, 5)
    b.fill(g)
    q = normal(g, (nh, b.nt, 128), F16)
    want, tol = ref.attention(b, q, True, 128 ** -0.5)
    o = torch.empty_like(q)
    first = None
    for _ in range(30):
        o.fill_(7.0)
        attend(pkg, ops.attention, b, q, o)
        first = o.clone() if first is None else first
        assert torch.equal(o, first)
    near(o, want, tol, "o")
    assert ops.attention.status() == 0


@pytest.mark.parametrize("n,kv,nkvh", [([1], [3000], 1), ([1, 1], [40, 9000], 2), ([30], [2500], 2), ([150, 20], [400, 6000], 1), ([1500], [1500], 2)])
def test_attention_paged_nan_queries(pkg, dev, ops, n, kv, nkvh):
    """A NaN in a query is that row's alone, and shows, in however many parts the row is computed; so does one in a key, in all rows
    that see it."""
    b = ref.Batch(dev, F16, n, kv, nkvh, 64, 16, seed=7)
    g = gen(dev, 7)
    b.fill(g)
    nh = 4 * nkvh
    q = normal(g, (nh, b.nt, 64), F16)
    want, tol = ref.attention(b, q, True, 0.125)
    bent = q.clone()
    for h in range(0, nh, 3):
        bent[h, :: 7, 5] = math.nan
    o = torch.zeros_like(q)
    attend(pkg, ops.attention, b, bent, o)
    hit = torch.isnan(bent).any(-1)
    assert bool(torch.isnan(o[hit]).all())
    near(o[~hit], want[~hit], tol[~hit], "the other rows")
    page, slot = b.slots(0, 3, 4)
    b.k_pages[page, 0, slot] = math.nan
    attend(pkg, ops.attention, b, q, o)
    sees = torch.zeros(nh, b.nt, dtype=torch.bool, device=dev)
    sees[:4, max(0, 3 - (kv[0] - n[0])): n[0]] = True
    assert bool(torch.isnan(o[sees]).all())
    near(o[~sees], want[~sees], tol[~sees], "the other rows")


def test_attention_paged_short_workspace(pkg, dev, ops):
    """Without one the operator says how much it wants (and Operator.launch gets it)."""
    b = ref.Batch(dev, F16, [1, 90], [5000, 100], 2, 128, 16, seed=8)
    g = gen(dev, 8)
    b.fill(g)
    q = normal(g, (8, b.nt, 128), F16)
    o, o2 = torch.zeros_like(q), torch.zeros_like(q)
    attend(pkg, ops.attention, b, q, o)
    ops.attention.launch(pkg.AttentionPagedArgs.of(q, b.k_pages, b.v_pages, o2, b.descriptor(pkg)))
    assert torch.equal(o, o2)


def test_large_strides_past_32_bits(pkg, dev, ops):
    """Pages more than 4 GB apart: offsets are 64-bit."""
    n, kv = [1, 40], [200, 300]
    ps, dh = 64, 128
    b = ref.Batch(dev, F16, n, kv, 1, dh, ps, seed=3, spare=1)
    step = 700 * 2 ** 20 // 2  # 700 MB between pages: the 13th ends beyond 8 GB
    buf = torch.empty((b.npages - 1) * step + ps * dh, dtype=F16, device=dev)
    b.k_pages = buf.as_strided((b.npages, 1, ps, dh), (step, ps * dh, dh, 1))
    assert (b.npages - 1) * step * 2 > 2 ** 32
    check_attention(pkg, dev, ops.attention, b, 4)
    qkv = normal(gen(dev, 2), (b.nt, 3, dh), F16)
    pos = torch.zeros(b.nt, dtype=torch.int32, device=dev).view(torch.uint32)  # position 0 turns nothing
    q_out = torch.empty(b.nt, 1, dh, dtype=F16, device=dev)
    ops.append.launch(pkg.KvAppendPagedArgs.of(q_out, qkv[:, :1], qkv[:, 1:2], qkv[:, 2:], b.k_pages, b.v_pages, pos, b.descriptor(pkg), THETA))
    for i, (m, l) in enumerate(zip(n, kv)):
        page, slot = b.slots(i, l - m, l)
        r = int(b.start[i])
        assert torch.equal(b.k_pages[page, :, slot], qkv[r: r + m, 1:2]) and torch.equal(b.v_pages[page, :, slot], qkv[r: r + m, 2:])


# ------------------------------------------------------------------------------------------------ a run of them together
@pytest.mark.parametrize("dt,norm", [(F16, False), (BF16, True)])
def test_steps_of_a_batch(pkg, dev, ops, dt, norm):
    """Prompts in chunks, then single tokens, sequences joining on the way: append and attend step after step, against the 64-bit
    forms over the whole history."""
    nh, nkvh, dh, ps = 8, 2, 64, 16
    steps = [[37, 0, 0], [20, 5, 0], [1, 130, 3], [1, 1, 1], [1, 1, 1]]
    total = [sum(s[i] for s in steps) for i in range(3)]
    b = ref.Batch(dev, dt, [0] * 3, total, nkvh, dh, ps, seed=1)
    g = gen(dev, 3)
    w = (1 + 0.3 * torch.randn(nh + nkvh, dh, generator=g, device=dev)).to(dt) if norm else None
    done = [0, 0, 0]
    for n in steps:
        rows = sum(n)
        qkv = normal(g, (rows, nh + 2 * nkvh, dh), dt)
        kv = [d + x for d, x in zip(done, n)]
        pos = torch.cat([torch.arange(d, e) for d, e in zip(done, kv)]).to(dev)
        b.n, b.kv, b.nt = n, kv, rows
        b.start = torch.tensor([sum(n[:i]) for i in range(4)])
        b.seq_start.copy_(b.start)
        b.kv_len.copy_(torch.tensor(kv))
        q, k, v = qkv[:, :nh], qkv[:, nh: nh + nkvh], qkv[:, nh + nkvh:]
        want = ref.rotate(qkv[:, : nh + nkvh].double(), pos, THETA, w, EPS)
        tol = ref.rotate_tolerance(qkv[:, : nh + nkvh].double(), pos, THETA, w, EPS, dt, want)
        ops.append.launch(pkg.KvAppendPagedArgs.of(q, q, k, v, b.k_pages, b.v_pages, pos.to(torch.uint32), b.descriptor(pkg), THETA, w, EPS))
        near(q, want[:, :nh], tol[:, :nh], "q")
        o = torch.empty(rows, nh, dh, dtype=dt, device=dev)
        attend(pkg, ops.attention, b, q.permute(1, 0, 2), o.permute(1, 0, 2))
        near(o.permute(1, 0, 2), *ref.attention(b, q.permute(1, 0, 2), True, dh ** -0.5), "o")
        done = kv
    assert ops.append.status() == 0 and ops.attention.status() == 0


def _weights(dev, cfg, norm):
    g = gen(dev, 11)
    qkv = (cfg.nh + 2 * cfg.nkvh) * cfg.dh
    w = {"w_norm1": (torch.rand(cfg.d, generator=g, device=dev) + 0.5).half(), "w_qkv": normal(g, (cfg.d, qkv), F16, 0.05),
         "w_o": normal(g, (cfg.nh * cfg.dh, cfg.d), F16, 0.05), "w_norm2": (torch.rand(cfg.d, generator=g, device=dev) + 0.5).half(),
         "w_gu": normal(g, (cfg.d, 2 * cfg.ffn), F16, 0.05), "w_down": normal(g, (cfg.ffn, cfg.d), F16, 0.05)}
    if norm:
        w["w_qk_norm"] = (torch.rand(cfg.nh + cfg.nkvh, cfg.dh, generator=g, device=dev) + 0.5).half()
    return w


@pytest.mark.parametrize("norm", [False, True])
def test_layer_over_a_paged_cache(pkg, dev, norm):
    """DecoderLayer.forward_paged on two requests, prompts then single tokens, against DecoderLayer.forward on each request's
    whole text: the last token's row is the same function of the same tokens.  Tolerance: the layer test's 2e-2 of the larger of
    1 and |value| / 4 (f16 rounding points of the ten operators; both sides round at the same places but the score order)."""
    layer_mod = importlib.import_module(graft.PKG_NAME + ".layer")
    cfg = layer_mod.LayerConfig(d=512, nh=8, nkvh=2, dh=64, ffn=1024)
    layer = layer_mod.DecoderLayer(cfg, _weights(dev, cfg, norm), 256, dev)
    texts = [normal(gen(dev, 21), (70, cfg.d), F16), normal(gen(dev, 22), (133, cfg.d), F16)]
    full = []
    for t in texts:
        full.append(layer.forward(t.clone(), torch.arange(len(t), dtype=torch.int32, device=dev).view(torch.uint32)).clone())
    ps = 16
    k_pages, v_pages = (torch.full((16, cfg.nkvh, ps, cfg.dh), math.nan, dtype=F16, device=dev) for _ in range(2))
    table = torch.randperm(16, generator=torch.Generator().manual_seed(1)).to(torch.int32)
    table = torch.stack([torch.cat([table[:5], table[5:9]]), torch.cat([table[5:14]])]).to(dev)
    done = [0, 0]
    for n in ([64, 100], [4, 32], [1, 1], [1, 0]):
        rows = torch.cat([t[d: d + x] for t, d, x in zip(texts, done, n)] + [torch.zeros(3, cfg.d, dtype=F16, device=dev)])  # three rows of nobody
        kv = [d + x for d, x in zip(done, n)]
        pos = torch.cat([torch.arange(d, e) for d, e in zip(done, kv)] + [torch.zeros(3, dtype=torch.int64)]).to(torch.int32).to(dev).view(torch.uint32)
        batch = pkg.PagedBatch(table, torch.tensor([0, n[0], sum(n)], dtype=torch.int32, device=dev), torch.tensor(kv, dtype=torch.int32, device=dev), max(n))
        out = layer.forward_paged(rows, pos, batch, k_pages, v_pages)
        for i, (d, e) in enumerate(zip(done, kv)):
            at = n[0] * i
            want = full[i][d:e].double()
            near(out[at: at + n[i]], want, 2e-2 * want.abs().div(4).clamp(min=1), f"request {i}, tokens {d}..{e}")
        done = kv
    assert layer.attention_paged.status() == 0 and layer.kv_append_paged.status() == 0


def test_layer_captured_step_after_a_larger_one(pkg, dev):
    """A captured step of single tokens goes on working after prompts have passed through the layer: its scratch is still there."""
    layer_mod = importlib.import_module(graft.PKG_NAME + ".layer")
    cfg = layer_mod.LayerConfig(d=512, nh=8, nkvh=2, dh=64, ffn=1024)
    layer = layer_mod.DecoderLayer(cfg, _weights(dev, cfg, False), 256, dev)
    ps = 16
    k_pages, v_pages = (normal(gen(dev, k), (80, cfg.nkvh, ps, cfg.dh), F16) for k in (1, 2))
    table = torch.arange(80, dtype=torch.int32, device=dev).view(2, 40)

    def step(n, kv):
        at = torch.cat([torch.arange(l - x, l) for x, l in zip(n, kv)])
        batch = pkg.PagedBatch(table, torch.tensor([0, n[0], sum(n)], dtype=torch.int32, device=dev), torch.tensor(kv, dtype=torch.int32, device=dev), max(n))
        return at.to(torch.int32).to(dev).view(torch.uint32), batch

    rows = normal(gen(dev, 3), (2, cfg.d), F16)
    x, (pos, batch) = rows.clone(), step([1, 1], [600, 513])
    want = layer.forward_paged(x, pos, batch, k_pages, v_pages).clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.forward_paged(x, pos, batch, k_pages, v_pages)
    keys, values = k_pages.clone(), v_pages.clone()
    for n, kv in (([100, 30], [130, 40]), ([1, 60], [20, 70])):
        p, b = step(n, kv)
        layer.forward_paged(normal(gen(dev, 4), (sum(n), cfg.d), F16), p, b, k_pages, v_pages)
    k_pages.copy_(keys)
    v_pages.copy_(values)
    junk = [torch.full((2 ** 20,), math.nan, device=dev) for _ in range(64)]  # takes what is free
    for _ in range(3):
        x.copy_(rows)
        graph.replay()
        assert torch.equal(out, want)
    assert len(junk) == 64 and layer.attention_paged.status() == 0


def test_streams_of_every_kind_of_device(pkg, dev):
    """A queue named by an index, a torch device, a string or nothing is torch's current stream."""
    side = torch.cuda.Stream(dev)
    for _ in range(2):
        for device in (None, 0, dev, torch.device("cuda"), "cuda:0"):
            assert pkg.TorchQueueAlloc(device).queue() == pkg.current_stream(device) == torch.cuda.current_stream().cuda_stream
            with torch.cuda.stream(side):
                assert pkg.TorchQueueAlloc(device).queue() == side.cuda_stream
        pkg.Rope(0)
