"""Batches that the paged operators have to report or to survive, beside those of test_gpu_paged.py."""
import math

import pytest
import torch

import paged_reference as ref
from test_gpu_paged import BF16, F16, THETA, attend, check_attention, gen, near, normal

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ kv_append_paged: the whole batch is looked at
@pytest.mark.parametrize("start,bad", [([3, 0], True),               # every row is in front of the first sequence, or behind the last
                                       ([0, 4, 2, 6], True),         # rows 2 and 3 are claimed twice
                                       ([0, 6, 6, 2, 6], True),      # a fall between sequences that own no row
                                       ([0, 6, 900, 6], True),       # past the step's rows, and back
                                       ([0, 2, 2, 6], False), ([2, 2, 6], False)])
@pytest.mark.parametrize("nt", [6, 40])
def test_kv_append_paged_reports_starts_that_fall(pkg, dev, start, bad, nt):
    op = pkg.KvAppendPaged(0)
    nseq, ps = len(start) - 1, 16
    k_pages, v_pages = (torch.full((nseq, 2, ps, 64), math.nan, dtype=F16, device=dev) for _ in range(2))
    ints = [torch.tensor(x, dtype=torch.int32, device=dev) for x in ([[i] for i in range(nseq)], start, [ps] * nseq)]
    qkv = normal(gen(dev, 1), (nt, 8, 64), F16)
    pos = torch.arange(nt, dtype=torch.int32, device=dev).view(torch.uint32)
    op.launch(pkg.KvAppendPagedArgs.of(qkv[:, :4].clone(), qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], k_pages, v_pages, pos, pkg.PagedBatch(*ints), THETA))
    assert op.status() == (pkg.PAGED_BAD_ROWS if bad else 0)


def test_kv_append_paged_reports_a_length_of_an_idle_sequence(pkg, dev):
    """As attention_paged does: kv_len beyond what the table maps, though none of the step's rows is the sequence's."""
    op = pkg.KvAppendPaged(0)
    n = 300
    k_pages, v_pages = (torch.zeros(2, 2, 16, 64, dtype=F16, device=dev) for _ in range(2))
    for at in (0, 150, n - 1):
        length = torch.zeros(n, dtype=torch.int32, device=dev)
        length[at] = 17
        start = torch.zeros(n + 1, dtype=torch.int32, device=dev)
        if at < n - 1:
            start[n], length[n - 1] = 2, 2  # two rows, the last sequence's
        qkv = normal(gen(dev, 1), (2, 8, 64), F16)
        pos = torch.arange(2, dtype=torch.int32, device=dev).view(torch.uint32)
        batch = pkg.PagedBatch(torch.zeros(n, 1, dtype=torch.int32, device=dev), start, length)
        op.launch(pkg.KvAppendPagedArgs.of(qkv[:, :4].clone(), qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], k_pages, v_pages, pos, batch, THETA))
        assert op.status() == pkg.PAGED_BAD_LENGTH
        op.status_reset()


# ------------------------------------------------------------------------------------------------ status words
@pytest.mark.parametrize("cls", ["KvAppendPaged", "AttentionPaged"])
def test_status_of_a_handle_made_on_a_busy_device(pkg, dev, cls):
    """What a launch on a stream of its own reports stays, although the default stream was busy when the handle was made: the
    words are clear before the handle is there, not some time after."""
    b = ref.Batch(dev, F16, [1], [20], 2, 64, 16, seed=1)
    b.fill(gen(dev, 1))
    b.page_table[0, 1] = b.npages
    qkv = normal(gen(dev, 2), (1, 8, 64), F16)
    pos = torch.zeros(1, dtype=torch.int32, device=dev).view(torch.uint32)
    o, ws, side = torch.zeros(4, 1, 64, dtype=F16, device=dev), torch.empty(64 << 20, dtype=torch.uint8, device=dev), torch.cuda.Stream(dev)

    def launch(op):
        with torch.cuda.stream(side):
            if cls == "KvAppendPaged":
                op.launch(pkg.KvAppendPagedArgs.of(qkv[:, :4], qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], b.k_pages, b.v_pages, pos, b.descriptor(pkg), THETA))
            else:
                attend(pkg, op, b, qkv[:, :4].permute(1, 0, 2), o, ws=ws)

    launch(getattr(pkg, cls)(0))  # a kernel's first launch may wait for the device
    torch.cuda.synchronize()
    torch.cuda._sleep(300_000_000)  # some 0.2 s of the default stream
    op = getattr(pkg, cls)(0)
    launch(op)
    assert op.status() == pkg.PAGED_BAD_PAGE
    op.status_reset()
    assert op.status() == 0


# ------------------------------------------------------------------------------------------------ work far apart
@pytest.mark.parametrize("n,past", [([300] + [0] * 3000 + [200], 300),                   # idle sequences between two chunks
                                    ([70] + [1] * 300 + [0] * 33 + [60, 0, 0, 80], 90),  # single tokens, which the tiles have nothing of
                                    ([0] * 200 + [1] + [0] * 5000 + [1], 2500),          # ... and single tokens far apart
                                    ([1] + [40] * 5 + [0] * 129 + [40] * 3 + [1] * 2, 700)])
def test_attention_paged_sequences_far_apart(pkg, dev, n, past):
    kv = [m + (past + 13 * i % 50 if m else 0) for i, m in enumerate(n)]
    check_attention(pkg, dev, pkg.AttentionPaged(0), ref.Batch(dev, F16, n, kv, 2, 64, 16, seed=4, pad=3), 4)


# ------------------------------------------------------------------------------------------------ parts that do not wait for one another
@pytest.mark.parametrize("n,kv,nkvh,nh,dh", [([40], [12000], 9, 36, 128), ([20, 30, 300], [9000, 9500, 9800], 3, 12, 128), ([33], [20000], 1, 8, 64),
                                             ([1, 700], [3000, 6000], 1, 4, 128)])
def test_attention_paged_units_whose_parts_do_not_wait(pkg, dev, n, kv, nkvh, nh, dh):
    """Units of many parts, joined by all their warps together when they meet, by the last to come when the others have left: bit
    for bit the same, from a patience that none outlasts through one that some do to the ordinary one."""
    op = pkg.AttentionPaged(0)
    b = ref.Batch(dev, BF16, n, kv, nkvh, dh, 16, seed=6)
    g = gen(dev, 6)
    b.fill(g)
    q = normal(g, (nh, b.nt, dh), BF16)
    want = torch.empty_like(q)
    ws = attend(pkg, op, b, q, want)
    near(want, *ref.attention(b, q, True, dh ** -0.5), "o")
    o = torch.empty_like(q)
    for patience in [0] * 30 + [500, 1000, 2000, 4000] * 15 + [100000]:
        op.set_patience(patience)
        o.fill_(7.0)
        ws.fill_(0xff)
        attend(pkg, op, b, q, o, ws=ws)
        assert torch.equal(o, want), patience
    assert op.status() == 0


def test_attention_paged_patience_is_bounded(pkg, dev):
    op = pkg.AttentionPaged(0)
    with pytest.raises(pkg.SchemeError):
        op.set_patience(10 ** 9 + 1)
    op.set_patience(10 ** 9)


# ------------------------------------------------------------------------------------------------ values that no score may meet
# Past and chunk by kernel: few rows, a few drafted tokens, tiles in one part, tiles of many parts.
SPECIAL = [([1, 1], [700, 40], 2), ([3, 2], [900, 40], 2), ([300, 20], [400, 50], 4), ([40, 30], [9000, 300], 4)]


def plain(b, i, q, scale, hidden=()):
    """Sequence i's rows over its slots but `hidden`, in doubles: ([nh, n, dh], tolerance as ref.attention derives it, slots a row sees)."""
    n, l, r0 = b.n[i], b.kv[i], int(b.start[i])
    page, slot = b.slots(i, 0, l)
    see = torch.arange(l, device=q.device)[None] <= torch.arange(l - n, l, device=q.device)[:, None]
    see[:, list(hidden)] = False
    out, tol = [], []
    for h in range(q.shape[0]):
        kv = h // (q.shape[0] // b.nkvh)
        k, v = b.k_pages[page, kv, slot].double().clone(), b.v_pages[page, kv, slot].double().clone()
        k[list(hidden)], v[list(hidden)] = 0, 0
        x = q[h, r0: r0 + n].double()
        size = (x.abs() @ k.abs().T * scale).amax(-1, keepdim=True)
        p = torch.softmax((x @ k.T * scale).masked_fill(~see, -math.inf), -1)
        o = p @ v
        move = ref.HALF_STEP[b.dt] + 2 * b.dh * 2.0 ** -23 * size + 2.0 ** -20
        out.append(o)
        tol.append(ref.HALF_STEP[b.dt] * o.abs() + (1 + ref.HALF_STEP[b.dt]) * (move * (p @ v.abs()) + l * ref.LEAST[b.dt] * v.abs().amax()) + ref.LEAST[b.dt])
    return torch.stack(out), torch.stack(tol), see


def special(pkg, dev, dt, case, positive=False):
    n, kv, nh = SPECIAL[case]
    b = ref.Batch(dev, dt, n, kv, 1, 64, 16, seed=case)
    g = gen(dev, case)
    b.fill(g)
    q = normal(g, (nh, b.nt, 64), dt)
    return b, (q.abs() + 0.1 if positive else q)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("case", [1, 2, 3])
def test_attention_paged_keys_of_later_tokens(pkg, dev, dt, value, case):
    """A key that only the sequence's last token sees shows in no other row, whatever it holds."""
    b, q = special(pkg, dev, dt, case)
    wants = [plain(b, i, q, 0.125) for i in range(2)]
    page, slot = b.slots(0, b.kv[0] - 1, b.kv[0])
    b.k_pages[page, :, slot] = value
    o = torch.zeros_like(q)
    attend(pkg, pkg.AttentionPaged(0), b, q, o)
    near(o[:, : b.n[0] - 1], wants[0][0][:, :-1], wants[0][1][:, :-1], "the rows in front")
    near(o[:, b.n[0]:], *wants[1][:2], "the other sequence")


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("case", [1, 2, 3])
def test_attention_paged_values_of_later_tokens(pkg, dev, dt, value, case):
    """A value of the last token's that is no number shows in the rows that see it, in no other sequence, and in no unit of rows in
    front of which ends before its block of keys (rows that share a block with it are documented to take it with a weight of zero)."""
    b, q = special(pkg, dev, dt, case)
    wants = [plain(b, i, q, 0.125) for i in range(2)]
    page, slot = b.slots(0, b.kv[0] - 1, b.kv[0])
    b.v_pages[page, :, slot] = value
    o = torch.zeros_like(q)
    attend(pkg, pkg.AttentionPaged(0), b, q, o)
    assert not torch.isfinite(o[:, b.n[0] - 1]).any()
    near(o[:, b.n[0]:], *wants[1][:2], "the other sequence")
    unit = 2 * (128 // q.shape[0])  # tokens of two tiles, the heads sharing one kv head
    for t0 in range(0, b.n[0] if case > 1 else 0, unit):
        if b.kv[0] - b.n[0] + t0 + unit <= (b.kv[0] - 1) // 128 * 128:
            near(o[:, t0: t0 + unit], wants[0][0][:, t0: t0 + unit], wants[0][1][:, t0: t0 + unit], f"tokens from {t0} on")


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("case", [0, 1, 2, 3])
@pytest.mark.parametrize("hidden", ["first", "some", "most"])
def test_attention_paged_scores_of_minus_infinity(pkg, dev, dt, case, hidden):
    """Keys of -inf against positive queries weigh nothing: the first blocks of a row entirely, single ones, all but a few."""
    b, q = special(pkg, dev, dt, case, positive=True)
    l = b.kv[0]
    past = l - b.n[0]
    which = {"first": range(0, min(257, past)), "some": range(0, l, 3), "most": [s for s in range(l) if s % 97 or s > past]}[hidden]
    want, tol, see = plain(b, 0, q, 0.125, which)
    page, slot = b.slots(0, 0, l)
    b.k_pages[page[list(which)], :, slot[list(which)]] = -math.inf
    o = torch.zeros_like(q)
    attend(pkg, pkg.AttentionPaged(0), b, q, o)
    rows = see.any(-1)
    near(o[:, : b.n[0]][:, rows], want[:, rows], tol[:, rows], "o")
    near(o[:, b.n[0]:], *plain(b, 1, q, 0.125)[:2], "the other sequence")


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("case", [0, 1, 2, 3])
def test_attention_paged_scores_of_infinity(pkg, dev, dt, case):
    """A score of +inf makes its row NaN, as the formula does (infinity less infinity), in however many parts; no other row."""
    b, q = special(pkg, dev, dt, case, positive=True)
    wants = [plain(b, i, q, 0.125) for i in range(2)]
    at = b.kv[0] - b.n[0] // 2 - 1  # the later half of the new tokens see it
    page, slot = b.slots(0, at, at + 1)
    b.k_pages[page, :, slot] = math.inf
    o = torch.zeros_like(q)
    attend(pkg, pkg.AttentionPaged(0), b, q, o)
    sees = wants[0][2][:, at]
    assert bool(torch.isnan(o[:, : b.n[0]][:, sees]).all())
    near(o[:, : b.n[0]][:, ~sees], wants[0][0][:, ~sees], wants[0][1][:, ~sees], "rows in front of it")
    near(o[:, b.n[0]:], *wants[1][:2], "the other sequence")


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("case", [0, 1, 2, 3])
def test_attention_paged_infinite_values(pkg, dev, dt, case):
    """An infinite value that all rows see with some weight makes its column infinite in all of them, and no other column."""
    b, q = special(pkg, dev, dt, case)
    q = q * 0.25  # scores of a fraction: no weight rounds to zero
    want, tol, see = plain(b, 0, q, 0.125)
    page, slot = b.slots(0, 5, 6)
    b.v_pages[page, :, slot, 7] = math.inf
    b.v_pages[page, :, slot, 9] = -math.inf
    o = torch.zeros_like(q)
    attend(pkg, pkg.AttentionPaged(0), b, q, o)
    got = o[:, : b.n[0]]
    assert bool((got[..., 7] == math.inf).all()) and bool((got[..., 9] == -math.inf).all())
    rest = [c for c in range(64) if c not in (7, 9)]
    near(got[..., rest], want[..., rest], tol[..., rest], "the other columns")


def test_operands_of_the_host_are_refused_beside_those_of_the_device(pkg, dev):
    b = ref.Batch(dev, F16, [1], [20], 2, 64, 16, seed=1)
    b.fill(gen(dev, 1))
    q, ws = normal(gen(dev, 2), (4, 1, 64), F16), torch.empty(64 << 20, dtype=torch.uint8, device=dev)
    op, o = pkg.AttentionPaged(0), torch.zeros(4, 1, 64, dtype=F16, device=dev)
    attend(pkg, op, b, q, o, ws=ws)
    want = o.clone()
    for bent in ((q.cpu(), b.k_pages, b.v_pages, o), (q, b.k_pages.cpu(), b.v_pages, o), (q, b.k_pages, b.v_pages.cpu(), o), (q, b.k_pages, b.v_pages, o.cpu())):
        with pytest.raises(ValueError, match="cuda:0 expected"):
            op.launch(pkg.AttentionPagedArgs.of(*bent, b.descriptor(pkg)), ws)
    for short in (ws.cpu(), ws[::2]):
        with pytest.raises(ValueError, match="workspace"):
            op.launch(pkg.AttentionPagedArgs.of(q, b.k_pages, b.v_pages, o, b.descriptor(pkg)), short)
    attend(pkg, op, b, q, o, ws=ws)
    assert torch.equal(o, want)


# ------------------------------------------------------------------------------------------------ workspaces of a stream of the caller's
def test_workspace_of_another_stream_is_not_handed_on_while_it_is_used(pkg, dev):
    """A launch on a queue of the caller's own, without a workspace: what the mirror allocates for it is that queue's, neither what
    the current stream may still be using nor, once the next launch has dropped it, what the current stream is given next."""
    b = ref.Batch(dev, F16, [1, 90], [5000, 100], 2, 128, 16, seed=8)
    g = gen(dev, 8)
    b.fill(g)
    q = normal(g, (8, b.nt, 128), F16)
    outs = [torch.zeros_like(q) for _ in range(3)]
    op = pkg.AttentionPaged(0)
    args = [pkg.AttentionPagedArgs.of(q, b.k_pages, b.v_pages, o, b.descriptor(pkg)) for o in outs]
    need = op.scheme(args[0])
    op.launch(args[0], torch.empty(need, dtype=torch.uint8, device=dev))
    for side in [torch.cuda.Stream(dev) for _ in range(6)]:  # some share a queue of the device's with the current stream: those wait anyway
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(100_000_000)
        queue = pkg.TorchQueueAlloc(dev, side.cuda_stream)
        free = torch.empty(need, dtype=torch.uint8, device=dev).data_ptr()  # the current stream's, until here
        op.launch(args[1], None, queue)
        assert op._last_ws.data_ptr() != free
        op.launch(args[2], None, queue)  # drops the first one's workspace
        mine = [torch.full((need,), 77, dtype=torch.uint8, device=dev) for _ in range(4)]  # of the current stream
        torch.cuda.synchronize()
        assert all(bool((x == 77).all()) for x in mine)
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
        del mine


def test_queues_of_every_kind_allocate(pkg, dev):
    side = torch.cuda.Stream(dev)
    for device in (None, 0, dev, "cuda:0"):
        for stream in (None, 0, side.cuda_stream, torch.cuda.current_stream().cuda_stream):
            mem = pkg.TorchQueueAlloc(device, stream).alloc(1000)
            assert mem.is_cuda and mem.numel() == 1000 and mem.get_device() == 0
