"""GPU parity of add and add_rows (the operators a caller chains around the decoder layer) against the CPU oracle.

Shapes follow the reference's tests: add over [2, 5632, 2048]-like tensors (operators/src/add/cuda/mod.rs), add_rows
with dst [b, m, n], src [k, n], idx [b, m] (operators/src/add_rows/cuda/mod.rs:205-290).  One f32 add per element and one
rounding: the f16 results are bit-exact.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def to_dev(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


@pytest.mark.parametrize("shape", [(2, 352, 2048), (7, 33), (5,), (3, 4, 5, 6, 8), (1, 1, 1)])
def test_add_contiguous(pkg, orc, synth, dev, shape):
    a = synth.normal(1, shape, 1.0).astype(np.float16)
    b = synth.normal(2, shape, 1.0).astype(np.float16)
    ad, bd = to_dev(a, dev), to_dev(b, dev)
    cd = torch.zeros_like(ad)
    pkg.Add(0).launch(pkg.AddArgs.of(cd, ad, bd))
    ref = orc.add(np.zeros_like(a), a, b)
    np.testing.assert_array_equal(cd.cpu().numpy().view(np.uint16), ref.view(np.uint16))


def test_add_strided_broadcast_and_in_place(pkg, orc, synth, dev):
    # a transposed, b broadcast along rows (stride 0), c a column slice of a wider buffer; then x += y in place
    a = synth.normal(3, (48, 64), 1.0).astype(np.float16)
    b = synth.normal(4, (1, 48), 1.0).astype(np.float16)
    cbuf = np.zeros((64, 96), np.float16)
    ad, bd, cd = to_dev(a, dev), to_dev(b, dev), to_dev(cbuf, dev)
    pkg.Add(0).launch(pkg.AddArgs.of(cd[:, 16:64], ad.t(), bd.expand(64, 48)))
    ref = cbuf.copy()
    orc.add(ref[:, 16:64], a.T, np.broadcast_to(b, (64, 48)))
    np.testing.assert_array_equal(cd.cpu().numpy().view(np.uint16), ref.view(np.uint16))
    x = synth.normal(5, (40, 4096), 1.0).astype(np.float16)
    y = synth.normal(6, (40, 4096), 1.0).astype(np.float16)
    xd = to_dev(x, dev)
    pkg.Add(0).launch(pkg.AddArgs.of(xd, xd, to_dev(y, dev)))
    np.testing.assert_array_equal(xd.cpu().numpy().view(np.uint16), orc.add(np.zeros_like(x), x, y).view(np.uint16))
    f = synth.normal(7, (9, 10), 1.0)
    fd = to_dev(f, dev)
    out = torch.zeros_like(fd)
    pkg.Add(0).launch(pkg.AddArgs.of(out, fd, fd))
    np.testing.assert_array_equal(out.cpu().numpy(), f + f)


def test_add_errors(pkg, dev):
    a = torch.zeros(4, 6, dtype=torch.float16, device=dev)
    op = pkg.Add(0)
    with pytest.raises(pkg.LaunchError) as e:
        op.launch(pkg.AddArgs.of(a, a, torch.zeros(4, 7, dtype=torch.float16, device=dev)))
    assert e.value.kind == pkg.SHAPE_MISMATCH
    with pytest.raises(pkg.LaunchError) as e:
        op.launch(pkg.AddArgs.of(a, a, torch.zeros(24, dtype=torch.float16, device=dev)))
    assert e.value.kind == pkg.RANK_MISMATCH
    with pytest.raises(pkg.LaunchError) as e:
        op.launch(pkg.AddArgs.of(a, a, torch.zeros(4, 6, dtype=torch.float32, device=dev)))
    assert e.value.kind == pkg.TYPE_MISMATCH
    with pytest.raises(pkg.LaunchError) as e:
        op.launch(pkg.AddArgs.of(a[:1].expand(4, 6), a, a))
    assert e.value.kind == pkg.SHAPE_NOT_SUPPORT and "Reducing" in e.value.info


@pytest.mark.parametrize("batch,m,n,k,idt", [(2, 7, 2048, 100, np.uint32), (1, 64, 4096, 128256 // 64, np.uint64), (3, 5, 40, 9, np.uint32)])
def test_add_rows(pkg, orc, synth, dev, batch, m, n, k, idt):
    dst = synth.normal(1, (batch, m, n), 1.0).astype(np.float16)
    src = synth.normal(2, (k, n), 1.0).astype(np.float16)
    idx = (synth.uniform01(3, (batch, m)) * k).astype(idt)
    dd, sd = to_dev(dst, dev), to_dev(src, dev)
    idd = to_dev(idx.view(np.int32 if idt == np.uint32 else np.int64), dev).view(torch.uint32 if idt == np.uint32 else torch.uint64)
    op = pkg.AddRows(0)
    op.launch(pkg.AddRowsArgs.of(dd, sd, idd))
    ref = orc.add_rows(dst.copy(), src, idx)
    np.testing.assert_array_equal(dd.cpu().numpy().view(np.uint16), ref.view(np.uint16))
    assert op.status() == 0


def test_add_rows_out_of_range_index_is_reported(pkg, synth, dev):
    dst = torch.ones(1, 3, 16, dtype=torch.float16, device=dev)
    src = torch.ones(4, 16, dtype=torch.float16, device=dev)
    idx = torch.tensor([[0, 9, 3]], dtype=torch.int32, device=dev).view(torch.uint32)
    op = pkg.AddRows(0)
    op.launch(pkg.AddRowsArgs.of(dst, src, idx))
    assert op.status() == 1  # the crate's CPU operator asserts idx < k; here the row is skipped and the status word set
    assert dst[0, 1].eq(1).all() and dst[0, 0].eq(2).all() and dst[0, 2].eq(2).all()


def test_add_rows_status_of_a_handle_made_on_a_busy_device(pkg, dev):
    """What a launch on a stream of its own reports stays, although the default stream was busy when the handle was made."""
    dst = torch.ones(1, 3, 16, dtype=torch.float16, device=dev)
    src = torch.ones(4, 16, dtype=torch.float16, device=dev)
    idx = torch.tensor([[0, 9, 3]], dtype=torch.int32, device=dev).view(torch.uint32)
    side = torch.cuda.Stream(dev)

    def launch(op):
        with torch.cuda.stream(side):
            op.launch(pkg.AddRowsArgs.of(dst, src, idx))

    launch(pkg.AddRows(0))  # a kernel's first launch may wait for the device
    torch.cuda.synchronize()
    torch.cuda._sleep(300_000_000)  # some 0.2 s of the default stream
    op = pkg.AddRows(0)
    launch(op)
    torch.cuda.synchronize()
    assert op.status() == 1
