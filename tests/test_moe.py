"""Refusals of the mixture-of-experts layer, without a GPU."""
import ctypes as C

import pytest
import torch

from flydsl_examples_b200 import _lib
from flydsl_examples_b200.moe_a16w16 import _POINTERS, _SCRATCH, _SIZES, _scratch_bytes, moe_a16w16


def args(**kw):
    a = _lib.MoeArgs()
    base = dict(x=4096, logits=4096, w13=4096, w2=4096, out=4096, tokens=4, hidden=64, inner=32, experts=8, ldx=64, logits_row=8, logits_col=1,
                w13_expert=64 * 64, w13_row=64, w2_expert=64 * 32, w2_row=32, ldo=64, top_k=2, renormalize=1, dtype=2, logits_dtype=1,
                workspace=4096, workspace_bytes=1 << 20)
    for key, v in {**base, **kw}.items():
        setattr(a, key, v)
    return a


BAD = [dict(tokens=0), dict(hidden=0), dict(inner=-8), dict(experts=0), dict(top_k=0), dict(top_k=9), dict(dtype=1), dict(dtype=4), dict(logits_dtype=0),
       dict(hidden=60), dict(inner=36, w2_row=36), dict(ldx=56), dict(ldx=68), dict(w13_row=56), dict(w13_row=68), dict(w2_row=24),
       dict(w13_expert=64 * 63), dict(w2_expert=64 * 31), dict(w13_expert=64 * 64 + 4), dict(ldo=63)]


def test_entry_points_refuse_before_any_device_work():
    lib = _lib.load()
    for bad in BAD:
        assert lib.b200_gemm_moe_a16w16(C.byref(args(**bad)), None) == -1, bad
        assert lib.b200_gemm_moe_workspace_bytes(C.byref(args(**bad))) == 0
    for bad in (dict(x=None), dict(logits=None), dict(w13=None), dict(w2=None), dict(out=None), dict(x=4104), dict(w13=4104), dict(w2=4098),
                dict(out=4097), dict(logits=4098)):
        assert lib.b200_gemm_moe_a16w16(C.byref(args(**bad)), None) == -1, bad
    for big in (dict(tokens=65), dict(experts=513)):
        assert lib.b200_gemm_moe_a16w16(C.byref(args(**big)), None) == -7
    for ws in (dict(workspace=None), dict(workspace=4100), dict(workspace_bytes=4096)):
        assert lib.b200_gemm_moe_a16w16(C.byref(args(**ws)), None) == -3
    # a list of experts, and h for every expert that four tokens can choose
    assert lib.b200_gemm_moe_workspace_bytes(C.byref(args())) == 4096 + 8 * 4 * 32 * 4
    assert lib.b200_gemm_moe_workspace_bytes(C.byref(args(tokens=1))) == 4096 + 2 * 1 * 32 * 4
    assert lib.b200_gemm_moe_a16w16(None, None) == -1
    for t, i, e, k in ((4, 32, 8, 2), (1, 32, 8, 2), (64, 2048, 512, 16)):  # the Python call's own sum
        assert _scratch_bytes(t, i, e, k) == lib.b200_gemm_moe_workspace_bytes(C.byref(args(
            tokens=t, inner=i, w2_row=i, w2_expert=64 * i, w13_expert=128 * i, experts=e, top_k=k)))
    assert _POINTERS.size + _SIZES.size + _SCRATCH.size + 8 == C.sizeof(_lib.MoeArgs)  # the byte string that the Python call passes


def test_structure_matches_the_header(tmp_path):
    import shutil
    import subprocess
    from pathlib import Path

    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no host C compiler")
    lines = ['printf("%zu\\n", sizeof(b200_gemm_moe_args));'] + [f'printf("%zu\\n", offsetof(b200_gemm_moe_args, {f}));' for f, _ in _lib.MoeArgs._fields_]
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "b200_gemm.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    inc = Path(__file__).resolve().parents[1] / "include"
    subprocess.run([cc, "-std=c99", f"-I{inc}", "-o", str(tmp_path / "s"), str(src)], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(_lib.MoeArgs)] + [getattr(_lib.MoeArgs, f).offset for f, _ in _lib.MoeArgs._fields_]


def test_python_refusals():
    bf = torch.bfloat16
    x, logits = torch.zeros(4, 64, dtype=bf), torch.zeros(4, 8)
    w13, w2 = torch.zeros(8, 64, 64, dtype=bf), torch.zeros(8, 64, 32, dtype=bf)
    with pytest.raises(ValueError, match="16-bit"):
        moe_a16w16(x.float(), logits, w13, w2, 2)
    with pytest.raises(ValueError, match="16-bit"):
        moe_a16w16(x, logits, w13.half(), w2, 2)
    with pytest.raises(ValueError, match="logits"):
        moe_a16w16(x, logits.double(), w13, w2, 2)
    with pytest.raises(ValueError, match="logits"):
        moe_a16w16(x, logits[:, :7], w13, w2, 2)
    with pytest.raises(ValueError, match="top_k"):
        moe_a16w16(x, logits, w13, w2, 9)
    with pytest.raises(ValueError, match="top_k"):
        moe_a16w16(x, logits, w13, w2, 0)
    with pytest.raises(ValueError, match="tokens"):
        moe_a16w16(torch.zeros(65, 64, dtype=bf), torch.zeros(65, 8), w13, w2, 2)
    with pytest.raises(ValueError, match="multiples of 8"):
        moe_a16w16(x[:, :60], logits, w13[:, :, :60], w2[:, :60], 2)
    with pytest.raises(ValueError, match="w2"):
        moe_a16w16(x, logits, w13, w2[:, :56], 2)
    with pytest.raises(ValueError, match="w13"):
        moe_a16w16(x, logits, w13.transpose(1, 2), w2, 2)
    with pytest.raises(ValueError, match="16-byte"):
        moe_a16w16(torch.zeros(4, 72, dtype=bf)[:, 4:68], logits, w13, w2, 2)
    with pytest.raises(ValueError, match="key"):
        moe_a16w16(x, logits, w13, w2, 2, user_kwargs={"tile_n": 16})
    with pytest.raises(AssertionError, match="out"):
        moe_a16w16(x, logits, w13, w2, 2, out=torch.zeros(4, 72, dtype=bf))
    with pytest.raises(AssertionError, match="CUDA"):
        moe_a16w16(x, logits, w13, w2, 2)


def test_calls_at_once_on_one_stream_have_scratch_of_their_own(monkeypatch):
    # A call is two launches, and the entry point runs without Python's lock: while it runs, another thread's call on the same
    # stream may come between the two. Here the second call is made from within the first one's.
    import threading

    from flydsl_examples_b200 import gemm_a16w16 as gemm, moe_a16w16 as module

    shared = gemm._Workspace(torch.device("cpu"))
    shared.ensure(_lib.COUNTER_BYTES + (1 << 20), torch.device("cpu"), None)
    monkeypatch.setattr(module, "_workspace_for", lambda *a: shared)
    monkeypatch.setattr(module, "raw_stream", lambda index: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: None)
    bf, running = torch.bfloat16, []

    def call(t):
        x, logits, w13, w2 = torch.zeros(t, 64, dtype=bf), torch.zeros(t, 8), torch.zeros(8, 64, 64, dtype=bf), torch.zeros(8, 64, 32, dtype=bf)
        need, sizes = module._call_plan(x.shape, x.stride(), x.dtype, logits.shape, logits.stride(), logits.dtype, w13.shape, w13.stride(), bf,
                                        w2.shape, w2.stride(), bf, x.shape, bf, 2, True, ())
        module._launch_moe(x, logits, w13, w2, torch.empty_like(x), need, sizes, 0)

    def entry(args, stream):
        a = _lib.MoeArgs.from_buffer_copy(args)
        running.append((a.workspace, a.workspace + a.workspace_bytes))
        if len(running) == 1:
            other = threading.Thread(target=call, args=(5,))
            other.start()
            other.join()
        return 0
    monkeypatch.setattr(module._lib, "fast", lambda name: entry)
    call(4)
    spans = running + [(shared.buf.data_ptr(), shared.buf.data_ptr() + shared.buf.numel())]  # what split-K GEMMs of the stream use
    assert len(spans) == 3
    for i, (lo, hi) in enumerate(spans):
        assert all(hi <= lo2 or hi2 <= lo for lo2, hi2 in spans[i + 1:])
