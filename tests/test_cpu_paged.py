"""What the paged operators and rope_norm refuse, through the C ABI without a device: every check of arguments comes before the
handle is looked at, so a null handle is enough (a call that passes all of them is answered with "null handle")."""
import ctypes
import os
import shutil
import subprocess

import pytest

P16 = 1 << 20  # a base pointer that is aligned and never followed


def L(pkg, dt, shape, strides=None):
    return pkg.TensorLayout.new_contiguous(dt, shape) if strides is None else pkg.TensorLayout(dt, shape, strides)


def batch(pkg, table=None, start=None, length=None, base=P16, max_seq=0):
    b = pkg.PagedBatch(table or L(pkg, pkg.I32, (3, 5)), start or L(pkg, pkg.I32, (4,)), length or L(pkg, pkg.I32, (3,)), max_seq)
    b.operands = tuple((*o[:-1], base) for o in b.operands)
    return b


def attention_args(pkg, q=None, k=None, v=None, o=None, b=None, mask=1, scale=0.125, base=P16):
    F16 = pkg.F16
    return pkg.AttentionPagedArgs(q or L(pkg, F16, (8, 7, 64)), base, k or L(pkg, F16, (10, 2, 16, 64)), base, v or L(pkg, F16, (10, 2, 16, 64)), base,
                                  o or L(pkg, F16, (8, 7, 64)), base, b or batch(pkg), mask, scale)


def append_args(pkg, b=None, base=P16, theta=1e4, eps=1e-5, w_base=None, **kw):
    F16 = pkg.F16
    d = {"q_out": L(pkg, F16, (7, 8, 64)), "q": L(pkg, F16, (7, 8, 64)), "k": L(pkg, F16, (7, 2, 64)), "v": L(pkg, F16, (7, 2, 64)),
         "k_pages": L(pkg, F16, (10, 2, 16, 64)), "v_pages": L(pkg, F16, (10, 2, 16, 64)), "p": L(pkg, pkg.U32, (7,)), "w": L(pkg, F16, (10, 64))}
    d.update(kw)
    return pkg.KvAppendPagedArgs(d["q_out"], base, d["q"], base, d["k"], base, d["v"], base, d["k_pages"], base, d["v_pages"], base, d["p"], base,
                                 d["w"], w_base, b or batch(pkg), eps, theta)


def norm_args(pkg, base=P16, theta=1e4, eps=1e-5, **kw):
    F16 = pkg.F16
    d = {"y": L(pkg, F16, (7, 10, 64)), "x": L(pkg, F16, (7, 10, 64)), "p": L(pkg, pkg.U32, (7,)), "w": L(pkg, F16, (10, 64))}
    d.update(kw)
    return pkg.RopeNormArgs(d["y"], base, d["x"], base, d["p"], base, d["w"], base, eps, theta)


def scheme(pkg, op, args):
    ws = ctypes.c_size_t(77)
    return getattr(pkg.lib(), f"ops_{op}_scheme")(None, args.byref(), ctypes.c_size_t(pkg.DYN_SIZE), ctypes.byref(ws))


def launch(pkg, op, args):
    if op == "rope_norm":
        return pkg.lib().ops_rope_norm_launch(None, args.byref(), None)
    return getattr(pkg.lib(), f"ops_{op}_launch")(None, args.byref(), None, ctypes.c_size_t(0), None)


def passes(pkg, op, args):
    """Nothing but the missing handle is wrong."""
    return launch(pkg, op, args) == pkg.ARGS_NOT_SUPPORT and "null handle" in pkg.last_error()


def test_the_calls_that_the_others_are_bent_from_pass(pkg):
    assert passes(pkg, "attention_paged", attention_args(pkg)) and scheme(pkg, "attention_paged", attention_args(pkg)) == 0
    assert passes(pkg, "kv_append_paged", append_args(pkg)) and scheme(pkg, "kv_append_paged", append_args(pkg)) == 0
    assert passes(pkg, "kv_append_paged", append_args(pkg, w_base=P16))
    assert passes(pkg, "rope_norm", norm_args(pkg))
    # any order of the cache's dims, a shared weight row, u32 arrays, padded rows
    assert passes(pkg, "attention_paged", attention_args(pkg, k=L(pkg, pkg.F16, (10, 2, 16, 64), (4096, 128, 256, 2))))
    assert passes(pkg, "rope_norm", norm_args(pkg, w=L(pkg, pkg.F32, (10, 64), (0, 4))))
    assert passes(pkg, "attention_paged", attention_args(pkg, b=batch(pkg, L(pkg, pkg.U32, (3, 5), (40, 4)), L(pkg, pkg.U32, (4,)), L(pkg, pkg.U32, (3,)))))


def test_attention_paged_refusals(pkg):
    F16, op = pkg.F16, "attention_paged"

    def bent(kind, **kw):
        assert scheme(pkg, op, attention_args(pkg, **kw)) == kind, (kw, pkg.last_error())
        assert launch(pkg, op, attention_args(pkg, **kw)) == kind, (kw, pkg.last_error())

    bent(pkg.RANK_NOT_SUPPORT, q=L(pkg, F16, (8, 448)))
    bent(pkg.RANK_NOT_SUPPORT, o=L(pkg, F16, (8, 448)))
    bent(pkg.RANK_NOT_SUPPORT, k=L(pkg, F16, (10, 2, 1024)))
    bent(pkg.RANK_NOT_SUPPORT, v=L(pkg, F16, (10, 2, 1024)))
    bent(pkg.RANK_NOT_SUPPORT, b=batch(pkg, table=L(pkg, pkg.I32, (15,))))
    bent(pkg.RANK_NOT_SUPPORT, b=batch(pkg, start=L(pkg, pkg.I32, (2, 2))))
    bent(pkg.RANK_NOT_SUPPORT, b=batch(pkg, length=L(pkg, pkg.I32, ())))
    bent(pkg.TYPE_NOT_SUPPORT, b=batch(pkg, table=L(pkg, pkg.I64, (3, 5))))
    bent(pkg.TYPE_NOT_SUPPORT, b=batch(pkg, length=L(pkg, pkg.F32, (3,))))
    bent(pkg.TYPE_NOT_SUPPORT, q=L(pkg, pkg.F32, (8, 7, 64)))
    bent(pkg.TYPE_MISMATCH, o=L(pkg, pkg.BF16, (8, 7, 64)))
    bent(pkg.TYPE_MISMATCH, v=L(pkg, pkg.BF16, (10, 2, 16, 64)))
    bent(pkg.SHAPE_MISMATCH, o=L(pkg, F16, (8, 6, 64)))
    bent(pkg.SHAPE_MISMATCH, o=L(pkg, F16, (4, 7, 64)))
    bent(pkg.SHAPE_MISMATCH, v=L(pkg, F16, (9, 2, 16, 64)))
    bent(pkg.SHAPE_MISMATCH, v=L(pkg, F16, (10, 2, 32, 64)))
    bent(pkg.SHAPE_MISMATCH, v=L(pkg, F16, (10, 2, 16, 128)))
    bent(pkg.SHAPE_MISMATCH, k=L(pkg, F16, (10, 3, 16, 64)), v=L(pkg, F16, (10, 3, 16, 64)))   # 8 heads over 3
    bent(pkg.SHAPE_MISMATCH, b=batch(pkg, start=L(pkg, pkg.I32, (3,))))
    bent(pkg.SHAPE_MISMATCH, b=batch(pkg, start=L(pkg, pkg.I32, (0,))))
    bent(pkg.SHAPE_NOT_SUPPORT, k=L(pkg, F16, (10, 2, 24, 64)), v=L(pkg, F16, (10, 2, 24, 64)))  # pages: powers of two
    bent(pkg.SHAPE_NOT_SUPPORT, k=L(pkg, F16, (10, 2, 4, 64)), v=L(pkg, F16, (10, 2, 4, 64)))
    bent(pkg.SHAPE_NOT_SUPPORT, q=L(pkg, F16, (8, 7, 136)), o=L(pkg, F16, (8, 7, 136)), k=L(pkg, F16, (10, 2, 16, 136)), v=L(pkg, F16, (10, 2, 16, 136)))
    bent(pkg.SHAPE_NOT_SUPPORT, q=L(pkg, F16, (8, 7, 60)), o=L(pkg, F16, (8, 7, 60)), k=L(pkg, F16, (10, 2, 16, 60)), v=L(pkg, F16, (10, 2, 16, 60)))
    bent(pkg.SHAPE_NOT_SUPPORT, q=L(pkg, F16, (258, 7, 64)), o=L(pkg, F16, (258, 7, 64)))
    bent(pkg.ARGS_NOT_SUPPORT, mask=2)

    def at_launch(kind, **kw):
        assert scheme(pkg, op, attention_args(pkg, **kw)) == 0, (kw, pkg.last_error())
        assert launch(pkg, op, attention_args(pkg, **kw)) == kind, (kw, pkg.last_error())

    D, S = pkg.DYN_SIZE, pkg.DYN_STRIDE
    at_launch(pkg.DYNAMIC_NOT_SUPPORT, q=L(pkg, F16, (8, D, 64), (S, 128, 2)))
    at_launch(pkg.DYNAMIC_NOT_SUPPORT, k=L(pkg, F16, (D, 2, 16, 64), (4096, 2048, 128, 2)))
    at_launch(pkg.DYNAMIC_NOT_SUPPORT, v=L(pkg, F16, (10, 2, 16, 64), (S, 2048, 128, 2)))
    at_launch(pkg.DYNAMIC_NOT_SUPPORT, b=batch(pkg, table=L(pkg, pkg.I32, (3, D), (S, 4))))
    at_launch(pkg.DYNAMIC_NOT_SUPPORT, b=batch(pkg, base=None))
    at_launch(pkg.DYNAMIC_NOT_SUPPORT, base=None)
    at_launch(pkg.DYNAMIC_NOT_SUPPORT, scale=pkg.DYN_F32)
    at_launch(pkg.STRIDES_NOT_SUPPORT, q=L(pkg, F16, (8, 7, 64), (896, 128, 4)))
    at_launch(pkg.STRIDES_NOT_SUPPORT, q=L(pkg, F16, (8, 7, 64), (904, 128, 2)))
    at_launch(pkg.STRIDES_NOT_SUPPORT, q=L(pkg, F16, (8, 7, 64), (896, -128, 2)))
    at_launch(pkg.STRIDES_NOT_SUPPORT, o=L(pkg, F16, (8, 7, 64), (898, 128, 2)))
    at_launch(pkg.STRIDES_NOT_SUPPORT, k=L(pkg, F16, (10, 2, 16, 64), (4096, 2048, 136, 2)))
    at_launch(pkg.STRIDES_NOT_SUPPORT, v=L(pkg, F16, (10, 2, 16, 64), (4096, -2048, 128, 2)))
    at_launch(pkg.STRIDES_NOT_SUPPORT, k=L(pkg, F16, (10, 2, 16, 64), (1 << 40, 2048, 128, 2)))
    at_launch(pkg.STRIDES_NOT_SUPPORT, base=P16 + 8)
    at_launch(pkg.STRIDES_NOT_SUPPORT, b=batch(pkg, base=P16 + 2))
    at_launch(pkg.STRIDES_NOT_SUPPORT, b=batch(pkg, table=L(pkg, pkg.I32, (3, 5), (40, 8))))
    at_launch(pkg.STRIDES_NOT_SUPPORT, b=batch(pkg, start=L(pkg, pkg.I32, (4,), (8,))))
    at_launch(pkg.SHAPE_NOT_SUPPORT, b=batch(pkg, table=L(pkg, pkg.I32, (3, 1 << 27))))  # 2^31 slots a sequence
    at_launch(pkg.SHAPE_NOT_SUPPORT, k=L(pkg, F16, (0, 2, 16, 64)), v=L(pkg, F16, (0, 2, 16, 64)))  # nothing to point a tensor map at
    # nothing to do is not an error, null pointers or not
    for kw in ({"q": L(pkg, F16, (8, 0, 64)), "o": L(pkg, F16, (8, 0, 64))},
               {"b": batch(pkg, L(pkg, pkg.I32, (0, 5)), L(pkg, pkg.I32, (1,)), L(pkg, pkg.I32, (0,)))}):
        assert launch(pkg, op, attention_args(pkg, **kw)) == 0, pkg.last_error()


def test_kv_append_paged_refusals(pkg):
    F16, op = pkg.F16, "kv_append_paged"

    def bent(kind, **kw):
        assert scheme(pkg, op, append_args(pkg, **kw)) == kind, (kw, pkg.last_error())
        assert launch(pkg, op, append_args(pkg, **kw)) == kind, (kw, pkg.last_error())

    for name in ("q", "q_out", "k", "v"):
        bent(pkg.RANK_NOT_SUPPORT, **{name: L(pkg, F16, (7, 512))})
        bent(pkg.TYPE_MISMATCH if name != "q" else pkg.TYPE_NOT_SUPPORT, **{name: L(pkg, pkg.F32, (7, 8 if "q" in name else 2, 64))})
        bent(pkg.SHAPE_MISMATCH, **{name: L(pkg, F16, (6, 8 if "q" in name else 2, 64))})
        bent(pkg.SHAPE_MISMATCH, **{name: L(pkg, F16, (7, 8 if "q" in name else 2, 32))})
    bent(pkg.SHAPE_MISMATCH, k=L(pkg, F16, (7, 3, 64)))
    bent(pkg.SHAPE_MISMATCH, p=L(pkg, pkg.U32, (8,)))
    bent(pkg.RANK_NOT_SUPPORT, p=L(pkg, pkg.U32, (7, 1)))
    bent(pkg.TYPE_NOT_SUPPORT, p=L(pkg, pkg.I32, (7,)))
    bent(pkg.RANK_NOT_SUPPORT, w=L(pkg, F16, (64,)), w_base=P16)
    bent(pkg.SHAPE_NOT_SUPPORT, k_pages=L(pkg, F16, (10, 2, 12, 64)), v_pages=L(pkg, F16, (10, 2, 12, 64)))
    wide = {n: L(pkg, F16, s) for n, s in {"q": (7, 8, 264), "q_out": (7, 8, 264), "k": (7, 2, 264), "v": (7, 2, 264), "k_pages": (10, 2, 16, 264),
                                           "v_pages": (10, 2, 16, 264)}.items()}
    bent(pkg.SHAPE_NOT_SUPPORT, **wide)

    def at_launch(kind, **kw):
        assert scheme(pkg, op, append_args(pkg, **kw)) == 0, (kw, pkg.last_error())
        assert launch(pkg, op, append_args(pkg, **kw)) == kind, (kw, pkg.last_error())

    at_launch(pkg.DYNAMIC_NOT_SUPPORT, theta=pkg.DYN_F32)
    at_launch(pkg.DYNAMIC_NOT_SUPPORT, eps=pkg.DYN_F32, w_base=P16)
    at_launch(pkg.DYNAMIC_NOT_SUPPORT, base=None)
    at_launch(pkg.DYNAMIC_NOT_SUPPORT, k=L(pkg, F16, (7, 2, 64), (pkg.DYN_STRIDE, 128, 2)))
    at_launch(pkg.STRIDES_NOT_SUPPORT, q_out=L(pkg, F16, (7, 8, 64), (1032, 128, 2)))
    at_launch(pkg.STRIDES_NOT_SUPPORT, v=L(pkg, F16, (7, 2, 64), (256, 128, 4)))
    at_launch(pkg.STRIDES_NOT_SUPPORT, base=P16 + 8)
    at_launch(pkg.STRIDES_NOT_SUPPORT, p=L(pkg, pkg.U32, (7,), (6,)))
    at_launch(pkg.SHAPE_MISMATCH, w=L(pkg, F16, (8, 64)), w_base=P16)
    at_launch(pkg.TYPE_NOT_SUPPORT, w=L(pkg, pkg.BF16, (10, 64)), w_base=P16)
    at_launch(pkg.STRIDES_NOT_SUPPORT, w=L(pkg, F16, (10, 64), (136, 2)), w_base=P16)
    at_launch(pkg.STRIDES_NOT_SUPPORT, w_base=P16 + 2)


def test_batch_of_host_tensors_is_refused(pkg):
    import torch
    table, start, length = torch.zeros(3, 5, dtype=torch.int32), torch.zeros(4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for arrays in ((table, L(pkg, pkg.I32, (4,)), L(pkg, pkg.I32, (3,))), (L(pkg, pkg.I32, (3, 5)), start, L(pkg, pkg.I32, (3,))),
                   (L(pkg, pkg.I32, (3, 5)), L(pkg, pkg.I32, (4,)), length)):
        with pytest.raises(ValueError, match="device tensors"):
            pkg.PagedBatch(*arrays)


def test_rope_norm_refusals(pkg):
    F16, op = pkg.F16, "rope_norm"

    def bent(kind, **kw):
        assert launch(pkg, op, norm_args(pkg, **kw)) == kind, (kw, pkg.last_error())

    bent(pkg.RANK_NOT_SUPPORT, x=L(pkg, F16, (7, 640)))
    bent(pkg.RANK_NOT_SUPPORT, w=L(pkg, F16, (64,)))
    bent(pkg.TYPE_MISMATCH, y=L(pkg, pkg.BF16, (7, 10, 64)))
    bent(pkg.TYPE_NOT_SUPPORT, p=L(pkg, pkg.I32, (7,)))
    bent(pkg.TYPE_NOT_SUPPORT, w=L(pkg, pkg.BF16, (10, 64)))
    bent(pkg.SHAPE_MISMATCH, y=L(pkg, F16, (7, 9, 64)))
    bent(pkg.SHAPE_MISMATCH, w=L(pkg, F16, (9, 64)))
    bent(pkg.SHAPE_MISMATCH, p=L(pkg, pkg.U32, (6,)))
    bent(pkg.DYNAMIC_NOT_SUPPORT, theta=pkg.DYN_F32)
    bent(pkg.DYNAMIC_NOT_SUPPORT, base=None)
    bent(pkg.DYNAMIC_NOT_SUPPORT, x=L(pkg, F16, (pkg.DYN_SIZE, 10, 64), (1280, 128, 2)))
    # what the chain of rms_norm and rope takes and this pass does not
    bent(pkg.ARGS_NOT_SUPPORT, x=L(pkg, pkg.F32, (7, 10, 64), (2560, 256, 2)), y=L(pkg, pkg.F32, (7, 10, 64), (2560, 256, 2)), w=L(pkg, pkg.F32, (10, 64)))
    bent(pkg.ARGS_NOT_SUPPORT, x=L(pkg, F16, (7, 10, 64), (1288, 128, 2)))
    bent(pkg.ARGS_NOT_SUPPORT, x=L(pkg, F16, (7, 10, 64), (1280, 128, 4)))
    bent(pkg.ARGS_NOT_SUPPORT, w=L(pkg, F16, (10, 64), (130, 2)))
    bent(pkg.ARGS_NOT_SUPPORT, x=L(pkg, F16, (7, 10, 60), (1280, 128, 2)), y=L(pkg, F16, (7, 10, 60), (1280, 128, 2)), w=L(pkg, F16, (10, 60), (128, 2)))
    assert "chain" in pkg.last_error()
    assert launch(pkg, op, norm_args(pkg, x=L(pkg, F16, (0, 10, 64)), y=L(pkg, F16, (0, 10, 64)), p=L(pkg, pkg.U32, (0,)))) == 0


def test_schedule_on_the_cpu(tmp_path):
    """The arithmetic that deals a batch to the CTAs (csrc/paged_schedule.h), compiled for the host, over random batches."""
    exe = str(tmp_path / "paged_schedule_check")
    src = os.path.join(os.path.dirname(os.path.abspath(__file__)), "paged_schedule_check.cc")
    built = subprocess.run([shutil.which("g++") or "g++", "-O2", "-std=c++17", src, "-o", exe], capture_output=True, text=True)
    assert built.returncode == 0, built.stderr
    ran = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert ran.returncode == 0 and "schedule ok" in ran.stdout, ran.stdout


@pytest.mark.parametrize("cls", ["KvAppendPaged", "AttentionPaged"])
def test_no_device_no_operator(pkg, cls):
    if pkg.device_count() > 0:
        pytest.skip("a CUDA device is present")
    with pytest.raises(pkg.SchemeError) as e:
        getattr(pkg, cls)(0)
    assert e.value.kind == pkg.EXECUTION_FAILED and "no CPU path" in e.value.info


class _Queue:
    """A queue that needs no device."""

    def queue(self):
        return 0


def _without_device(pkg, cls, calls):
    """An operator whose launches end in `calls`."""
    op = getattr(pkg, cls).__new__(getattr(pkg, cls))
    op.device, op._h = 0, None
    op._launch = lambda *a: calls.append(a) or 0
    return op


def test_operands_of_the_host_never_reach_a_kernel(pkg, monkeypatch):
    """A host tensor among the operands is refused where it would be launched; layouts and addresses are the caller's word."""
    import torch
    calls = []
    host = {name: torch.zeros(shape, dtype=dt) for name, shape, dt in (
        ("x", (7, 10, 64), torch.float16), ("q", (7, 8, 64), torch.float16), ("k", (7, 2, 64), torch.float16),
        ("pages", (10, 2, 16, 64), torch.float16), ("p", (7,), torch.uint32), ("w", (10, 64), torch.float16))}

    def bent(args, launch, cls):
        with pytest.raises(ValueError, match="cuda:0 expected"):
            launch(_without_device(pkg, cls, calls), args)

    F16 = pkg.F16
    lay = {"q": L(pkg, F16, (7, 8, 64)), "k": L(pkg, F16, (7, 2, 64)), "pages": L(pkg, F16, (10, 2, 16, 64)), "p": L(pkg, pkg.U32, (7,)), "w": L(pkg, F16, (10, 64))}
    operands = ["q", "q", "k", "k", "pages", "pages", "p", "w"]
    run = lambda op, args: op.launch(args, None, _Queue())  # noqa: E731
    for which in range(len(operands)):
        bases = [host[name] if i == which else P16 for i, name in enumerate(operands)]
        bent(pkg.KvAppendPagedArgs(*(x for name, base in zip(operands, bases) for x in (lay[name], base)), batch(pkg), 1e-5, 1e4), run, "KvAppendPaged")
    q, pages = L(pkg, F16, (8, 7, 64)), lay["pages"]
    operands = [(q, host["q"].transpose(0, 1)), (pages, host["pages"]), (pages, host["pages"]), (q, host["q"].transpose(0, 1))]
    for which in range(4):
        bent(pkg.AttentionPagedArgs(*(x for i, (layout, t) in enumerate(operands) for x in (layout, t if i == which else P16)), batch(pkg), 1, 0.125), run, "AttentionPaged")
    monkeypatch.setattr(pkg.lib(), "ops_rope_norm_launch", lambda *a: calls.append(a) or 0)
    x = L(pkg, F16, (7, 10, 64))
    operands = [(x, host["x"]), (x, host["x"]), (lay["p"], host["p"]), (lay["w"], host["w"])]
    for which in range(4):
        bent(pkg.RopeNormArgs(*(y for i, (layout, t) in enumerate(operands) for y in (layout, t if i == which else P16)), 1e-5, 1e4),
             lambda op, args: op.launch_norm(args, _Queue()), "Rope")
    with pytest.raises(ValueError, match="workspace"):
        _without_device(pkg, "AttentionPaged", calls).launch(attention_args(pkg), torch.zeros(1 << 20, dtype=torch.uint8), _Queue())
    assert not calls
    # addresses pass
    run(_without_device(pkg, "AttentionPaged", calls), attention_args(pkg))
    run(_without_device(pkg, "KvAppendPaged", calls), append_args(pkg))
    _without_device(pkg, "Rope", calls).launch_norm(norm_args(pkg), _Queue())
    assert len(calls) == 3


def test_schedule_of_sparse_batches_on_the_cpu(tmp_path):
    """Sequences without work on a line are passed over in runs."""
    exe = str(tmp_path / "paged_schedule_sparse_check")
    src = os.path.join(os.path.dirname(os.path.abspath(__file__)), "paged_schedule_sparse_check.cc")
    built = subprocess.run([shutil.which("g++") or "g++", "-O2", "-std=c++17", src, "-o", exe], capture_output=True, text=True)
    assert built.returncode == 0, built.stderr
    ran = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert ran.returncode == 0 and "schedule ok" in ran.stdout, ran.stdout


def test_schedule_of_launches_on_the_cpu(tmp_path):
    """The lines as a launch makes them: slots, counters and marks are nobody's twice."""
    exe = str(tmp_path / "paged_schedule_launch_check")
    src = os.path.join(os.path.dirname(os.path.abspath(__file__)), "paged_schedule_launch_check.cc")
    built = subprocess.run([shutil.which("g++") or "g++", "-O2", "-std=c++17", "-Wall", src, "-o", exe], capture_output=True, text=True)
    assert built.returncode == 0, built.stderr
    ran = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert ran.returncode == 0 and "schedule ok" in ran.stdout, ran.stdout


@pytest.mark.parametrize("rows,nseq,nkvh,fits", [(7, 3, 2, True), (1 << 20, 1 << 20, 8, True), (1 << 28, 1 << 28, 2, False), (1 << 29, 1, 128, False), (1, 1 << 27, 8, True)])
def test_attention_paged_refuses_more_units_than_a_line_holds(pkg, rows, nseq, nkvh, fits):
    """The device would find that they do not fit, write nothing and blame the batch."""
    F16, I32 = pkg.F16, pkg.I32
    q, kv = L(pkg, F16, (128, rows, 8)), L(pkg, F16, (10, nkvh, 16, 8))
    b = batch(pkg, L(pkg, I32, (nseq, 5)), L(pkg, I32, (nseq + 1,)), L(pkg, I32, (nseq,)))
    args = attention_args(pkg, q=q, o=q, k=kv, v=kv, b=b)
    if fits:
        assert passes(pkg, "attention_paged", args)
    else:
        assert launch(pkg, "attention_paged", args) == pkg.SHAPE_NOT_SUPPORT and "units" in pkg.last_error(), pkg.last_error()


def test_batch_of_a_negative_max_seq_is_refused(pkg):
    for wrong in (-1, 1 << 64):
        with pytest.raises(ValueError, match="max_seq"):
            batch(pkg, max_seq=wrong)


def test_argument_structs_are_those_of_the_header(pkg, tmp_path):
    """What the Python mirror packs by hand, read back by code that was compiled against the header."""
    lib = str(tmp_path / "libpaged_structs_check.so")
    src = os.path.join(os.path.dirname(os.path.abspath(__file__)), "paged_structs_check.cc")
    built = subprocess.run([shutil.which("g++") or "g++", "-O1", "-std=c++17", "-Wall", "-shared", "-fPIC", src, "-o", lib], capture_output=True, text=True)
    assert built.returncode == 0, built.stderr
    read = ctypes.CDLL(lib)
    bases = iter(range(0x1000, 0x100000, 0x1000))

    def field(name, dt, rank):
        base = next(bases)
        shape, strides = tuple(base + i for i in range(rank)), tuple(-base - i for i in range(rank))
        line = f"{name} dt {dt} shape {' '.join(map(str, shape))} strides {' '.join(map(str, strides))} base {base:x}"
        return pkg.TensorLayout(dt, shape, strides), base, line

    def check(function, make, names, tail, with_batch):
        fields = [field(name, dt, rank) for name, dt, rank in names]
        flat = [x for layout, base, _ in fields for x in (layout, base)]
        lines = [line for _, _, line in fields]
        more = []
        if with_batch:
            arrays = [field(name, pkg.U32, rank) for name, rank in (("page_table", 2), ("seq_start", 1), ("kv_len", 1))]
            b = pkg.PagedBatch(*(layout for layout, _, _ in arrays), 123456789012345)
            b.operands = tuple((*o[:-1], base) for o, (_, base, _) in zip(b.operands, arrays))
            more, lines = [b], lines + [line for _, _, line in arrays] + ["max_seq 123456789012345"]
        args = make(*flat, *more)
        front = 32  # an operand: u32 dt, u32 ndim, two pointers; its base
        size = len(names) * front + (3 * front + 8 if with_batch else 0) + 8
        fn = getattr(read, function)
        fn.restype = ctypes.c_char_p
        fn.argtypes = [ctypes.c_void_p]
        assert fn(args.byref()).decode().splitlines() == lines + [f"{tail} size {size}"]

    F16, BF16 = pkg.F16, pkg.BF16
    check("read_rope_norm", lambda *a: pkg.RopeNormArgs(*a, 0.25, 512.0), [("y", F16, 3), ("x", F16, 3), ("p", pkg.U64, 1), ("w", pkg.F32, 2)],
          "epsilon 0.25 theta 512", False)
    check("read_kv_append_paged", lambda *a: pkg.KvAppendPagedArgs(*a, 0.25, 512.0),
          [("q_out", F16, 3), ("q", F16, 3), ("k", BF16, 3), ("v", F16, 3), ("k_pages", BF16, 4), ("v_pages", F16, 4), ("p", pkg.U32, 1), ("w", F16, 2)],
          "epsilon 0.25 theta 512", True)
    check("read_attention_paged", lambda *a: pkg.AttentionPagedArgs(*a, 1, 0.125),
          [("q", F16, 3), ("k_pages", BF16, 4), ("v_pages", F16, 4), ("o", BF16, 3)], "mask 1 scale 0.125", True)


@pytest.mark.parametrize("tp", [1, 2, 4])
def test_norm_weights_of_the_heads_are_cut_with_them(pkg, tp):
    """Every head of a rank's shard has the weights that it has in the whole layer."""
    import importlib

    import numpy as np

    import __graft_entry__ as graft
    layer = importlib.import_module(graft.PKG_NAME + ".layer")
    nh, nkvh, dh, d, ffn = 12, 4, 8, 6, 16
    cfg = layer.LayerConfig(d=d, nh=nh, nkvh=nkvh, dh=dh, ffn=ffn)
    heads = np.arange(nh + 2 * nkvh, dtype=np.float32)
    w = {"w_norm1": np.ones(d), "w_norm2": np.ones(d), "w_qkv": np.repeat(heads, dh)[None].repeat(d, 0), "w_o": np.ones((nh * dh, d)),
         "w_gu": np.ones((d, 2 * ffn)), "w_down": np.ones((ffn, d)), "w_qk_norm": np.repeat(heads[: nh + nkvh, None], dh, 1)}
    seen = []
    for rank in range(tp):
        cut = layer.shard_weights(w, rank, tp, cfg)
        n = (nh + nkvh) // tp
        assert cut["w_qk_norm"].shape == (n, dh)
        of_columns = cut["w_qkv"][0].reshape(-1, dh)[:n]
        assert np.array_equal(of_columns, cut["w_qk_norm"])
        seen += cut["w_qk_norm"][:, 0].tolist()
    assert sorted(seen) == heads[: nh + nkvh].tolist()
