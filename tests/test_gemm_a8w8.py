"""Refusals, policy and structures of the 8-bit product, without a GPU."""
import ctypes as C
import struct

import pytest
import torch

from flydsl_examples_b200 import _lib, gemm_a8w8 as module
from flydsl_examples_b200.gemm_a8w8 import gemm_a8w8, heuristic_a8w8, linear_a8w8, plan, quantize_a8

E4 = torch.float8_e4m3fn


def zeros8(r, c):
    return torch.zeros(r, c, dtype=torch.uint8).view(E4)


def args8(**kw):
    a = _lib.Args8()
    base = dict(a=4096, b=8192, a_scale=4096, b_scale=4096, out=4096, m=256, n=256, k=256, lda=256, ldb=256, ldo=256, sa_row=1, sa_kb=256,
                sb_col=1, sb_kb=2, a_trans=0, b_trans=1, a_dtype=4, b_dtype=5, a_block=0, b_block=1, out_dtype=2)
    pol = {k: kw.pop(k) for k in list(kw) if k in ("tile_n", "cta_group", "split_k", "swap_ab", "stages", "stream_k", "loader", "tile_k")}
    for key, v in {**base, **kw}.items():
        setattr(a, key, v)
    for key, v in {"tile_n": 128, "cta_group": 1, **pol}.items():
        setattr(a.policy, key, v)
    return a


def query(**kw):
    pl = _lib.Plan()
    return _lib.load().b200_gemm_a8w8_plan_query(C.byref(args8(**kw)), C.byref(pl)), pl


def test_plan_and_bad_policies():
    rc, pl = query()
    assert rc == 0 and (pl.tile_m, pl.tile_n, pl.tiles_p, pl.tiles_q, pl.tile_k) == (128, 128, 2, 2, 128)
    rc, pl = query(tile_n=256, cta_group=2)
    assert rc == 0 and pl.tile_m == 256 and pl.tmem_cols == 512 and pl.smem_bytes <= 227 * 1024
    for bad in (dict(tile_n=48), dict(tile_n=256), dict(tile_n=64, cta_group=2), dict(tile_n=128, cta_group=2, split_k=2), dict(stages=3),
                dict(stream_k=1), dict(loader=1), dict(tile_k=64), dict(tile_n=64, b_trans=0), dict(tile_n=128, cta_group=2, b_trans=0)):
        assert query(**bad)[0] == -2, bad
    for bad in (dict(m=0), dict(k=-1), dict(a_dtype=2), dict(b_dtype=0), dict(out_dtype=4), dict(lda=128), dict(ldb=100), dict(ldo=255)):
        assert query(**bad)[0] == -1, bad
    assert query(m=1 << 31)[0] == -7
    # a cluster split is a power of two and no larger than the K blocks or the tile's columns
    assert query(tile_n=64, split_k=7, k=512, lda=512, ldb=512)[1].cluster_split == 4
    assert query(tile_n=16, split_k=16, k=8192, lda=8192, ldb=8192)[1].cluster_split == 16
    assert query(tile_n=16, split_k=16)[1].cluster_split == 2


def test_exponent_tiles_plan_and_refusals():
    both = dict(a_block=2, b_block=2, sa_kb=2, sb_kb=2)
    rc, pl = query(**both)
    assert rc == 0 and (pl.tile_n, pl.tmem_cols, pl.tiles_p, pl.tiles_q) == (128, 512, 2, 2) and pl.smem_bytes <= 227 * 1024
    for layout in (dict(b_trans=0), dict(a_trans=1, b_trans=0), dict(a_trans=1)):
        rc, pl = query(**both, tile_n=256, cta_group=2, **layout)
        assert rc == 0 and pl.tile_m == 256 and pl.tmem_cols == 512 and pl.smem_bytes <= 227 * 1024
    for bad in (dict(tile_n=64), dict(tile_n=16), dict(tile_n=128, cta_group=2), dict(split_k=2), dict(swap_ab=1)):
        assert query(**both, **bad)[0] == -2, bad
    for bad in (dict(a_block=2), dict(b_block=2), dict(a_block=3), dict(b_block=-1), dict(a_block=2, b_block=0)):
        assert query(**bad)[0] == -1, bad
    lib = _lib.load()
    for bad in (dict(a_scale=4104), dict(b_scale=4100), dict(sa_row=-1), dict(sb_kb=-1)):
        assert lib.b200_gemm_a8w8(C.byref(args8(**{**both, **bad})), None) == -1, bad
    assert lib.b200_gemm_a8w8(C.byref(args8(**{**both, "sa_row": 1 << 28})), None) == -7


def test_sequences_of_calls():
    lib = _lib.load()
    run = lambda *words: lib.b200_gemm_sequence(struct.pack(f"@{len(words)}q", *words), None)  # noqa: E731
    assert run(0) == 0 and run(4, 0) == -1 and run(-1, 0) == -1 and lib.b200_gemm_sequence(None, None) == -1
    quant = bytes(_lib.QuantizeArgs(rows=0, cols=8, in_dtype=1, out_dtype=4, mode=1))
    assert lib.b200_gemm_sequence(struct.pack("@q", 2) + quant + struct.pack("@q", 0), None) == 0
    bad = bytes(args8(m=0))
    assert lib.b200_gemm_sequence(struct.pack("@q", 2) + quant + struct.pack("@q", 1) + bad + struct.pack("@q", 0), None) == -1
    assert lib.b200_gemm_sequence(struct.pack("@q", 3) + bytes(_lib.ReduceArgs(rows=1, cols=4)) + struct.pack("@q", 0), None) == -1
    # the records that the linear layer packs
    for record, st in ((module._QUANT_RECORD, _lib.QuantizeArgs), (module._GEMM_RECORD, _lib.Args8), (module._REDUCE_RECORD, _lib.ReduceArgs)):
        assert struct.calcsize("@" + record) == 8 + C.sizeof(st)


def test_tiling_of_products_with_exponent_tiles():
    for sms in (148, 74, 1):
        for m, n, k in ((1, 1, 1), (300, 5000, 256), (1024, 2048, 4096), (2048, 4096, 4096), (8192, 8192, 8192)):
            tile, stages, split, group, swap, cg, *rest = module._packed_policy(m, n, k, sms)
            assert (tile, cg) in ((128, 1), (256, 2)) and (stages, split, swap) == (0, 1, 0) and not any(rest) and len(rest) == 10
    assert module._packed_policy(8192, 8192, 8192, 148)[0] == 256 and module._packed_policy(16, 4096, 4096, 148)[0] == 128


def test_entry_points_refuse_before_any_device_work():
    lib = _lib.load()
    for bad in (dict(a=None), dict(b_scale=None), dict(out=None), dict(a=4100), dict(b=8200), dict(lda=264), dict(a_scale=4098), dict(out=4097),
                dict(bias=4096, bias_dtype=0), dict(bias=4097, bias_dtype=2)):
        assert lib.b200_gemm_a8w8(C.byref(args8(**bad)), None) == -1, bad
    assert lib.b200_gemm_a8w8(None, None) == -1

    def quant(**kw):
        q = _lib.QuantizeArgs()
        base = dict(x=4096, rows=4, cols=64, ldx=64, in_dtype=2, out_dtype=4, mode=1, q_row=4096, ldq_row=64, s_row=4096, sr_row=1, sr_group=4)
        for key, v in {**base, **kw}.items():
            setattr(q, key, v)
        return lib.b200_gemm_quantize_a8(C.byref(q), None)
    for bad in (dict(rows=-1), dict(in_dtype=4), dict(out_dtype=2), dict(mode=0), dict(mode=5), dict(x=None), dict(ldx=63), dict(x=4097),
                dict(q_row=None), dict(s_row=None), dict(ldq_row=63), dict(mode=2), dict(mode=3), dict(colsum=4096, colsum_ld=64), dict(packed=2), dict(packed=-1)):
        assert quant(**bad) == -1, bad
    assert quant(rows=0) == 0 and quant(cols=0) == 0 and lib.b200_gemm_quantize_a8(None, None) == -1


def test_structures_match_the_header(tmp_path):
    import shutil
    import subprocess
    from pathlib import Path

    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no host C compiler")
    pairs = (("b200_gemm_a8w8_args", _lib.Args8), ("b200_gemm_quantize_args", _lib.QuantizeArgs),
             ("b200_gemm_reduce_args", _lib.ReduceArgs))
    lines, want = [], []
    for name, st in pairs:
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(C.sizeof(st))
        tail = {_lib.Args8: module._SIZES.size + 8, _lib.QuantizeArgs: module._QUANT_SIZES.size}.get(st)
        if tail is not None:
            assert module._POINTERS.size + tail == C.sizeof(st)  # the byte string that the Python calls pass
        for field, _ in st._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(st, field).offset)
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "b200_gemm.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    inc = Path(__file__).resolve().parents[1] / "include"
    subprocess.run([cc, "-std=c99", f"-I{inc}", "-o", str(tmp_path / "s"), str(src)], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == want


def test_python_refusals():
    a, b = zeros8(32, 256), zeros8(64, 256).t()
    sa, sb = torch.ones(32, 2), torch.ones(2, 1)
    with pytest.raises(ValueError, match="layout"):
        gemm_a8w8(a, sa, b, sb, layout="xx")
    with pytest.raises(ValueError, match="float8"):
        gemm_a8w8(torch.zeros(32, 256), sa, b, sb)
    with pytest.raises(ValueError, match="a_scale"):
        gemm_a8w8(a, torch.ones(32, 3), b, sb)
    with pytest.raises(ValueError, match="a_scale"):
        gemm_a8w8(a, torch.ones(32, 2, dtype=torch.float64), b, sb)
    with pytest.raises(ValueError, match="b_scale"):
        gemm_a8w8(a, sa, b, torch.ones(2, 3))
    with pytest.raises(ValueError, match="16-byte"):
        gemm_a8w8(zeros8(32, 264)[:, :250], torch.ones(32, 2), zeros8(64, 256)[:, :250].t(), sb)
    with pytest.raises(ValueError, match="A does not satisfy"):
        gemm_a8w8(a, sa, b, sb, layout="tt")
    with pytest.raises(ValueError, match="output dtype"):
        gemm_a8w8(a, sa, b, sb, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="bias"):
        gemm_a8w8(a, sa, b, sb, bias=torch.zeros(64, dtype=torch.float64))
    with pytest.raises(ValueError, match="policy key"):
        gemm_a8w8(a, sa, b, sb, user_kwargs={"stages": 3})
    with pytest.raises(ValueError, match="tile_n"):
        gemm_a8w8(a, sa, b, sb, user_kwargs={"swap_ab": True})
    with pytest.raises(AssertionError):
        gemm_a8w8(a, sa, zeros8(64, 128).t(), sb)
    with pytest.raises(AssertionError):
        gemm_a8w8(a, sa, b, sb, out=torch.zeros(32, 63, dtype=torch.bfloat16))
    with pytest.raises(AssertionError, match="CUDA"):
        gemm_a8w8(a, sa, b, sb)
    x = torch.zeros(4, 256)
    with pytest.raises(ValueError, match="group"):
        quantize_a8(x, "rows")
    with pytest.raises(ValueError, match="float8"):
        quantize_a8(x, "row", torch.int8)
    with pytest.raises(ValueError, match="takes"):
        quantize_a8(x.double())
    with pytest.raises(ValueError, match="row-major"):
        quantize_a8(torch.zeros(256, 4).t())
    with pytest.raises(AssertionError, match="matrix"):
        quantize_a8(torch.zeros(4))
    with pytest.raises(AssertionError, match="CUDA"):
        quantize_a8(x)
    with pytest.raises(AssertionError):
        linear_a8w8(x, torch.zeros(8, 128))
    with pytest.raises(AssertionError, match="CUDA"):
        linear_a8w8(x, torch.zeros(8, 256))


@pytest.mark.parametrize("m", [1, 16, 17, 64, 65, 200, 1000, 5000, 70000])
@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (7168, 2048), (4100, 4100), (100000, 130)])
@pytest.mark.parametrize("layout", ["nn", "nt", "tn", "tt"])
def test_heuristic_is_valid(m, n, k, layout):
    a_t, b_t = layout[0] == "t", layout[1] == "t"
    pol = heuristic_a8w8(m, n, k, a_t, b_t)
    up = lambda v: -(-v // 16) * 16  # noqa: E731
    rc, pl = query(m=m, n=n, k=k, lda=up(m if a_t else k), ldb=up(k if b_t else n), ldo=n, a_trans=int(a_t), b_trans=int(b_t),
                   tile_n=pol["tile_n"], cta_group=pol["cta_group"], split_k=pol["split_k"], swap_ab=int(pol["swap_ab"]))
    assert rc == 0 and pl.split_k == min(pol["split_k"], max(1, pl.split_k))


def test_plan_through_python():
    a, b = zeros8(8, 4096), zeros8(4096, 4096).t()
    got = plan(a, torch.ones(8, 32), b, torch.ones(32, 32))
    assert got["swap_ab"] == 1 and got["tile_n"] == 16 and got["cluster_split"] > 1


@pytest.mark.parametrize("sms", [148, 132, 74])
def test_a_split_keeps_all_its_clusters_running_at_once(sms):
    for m in (1, 8, 33, 64, 65, 128, 256, 700):
        for n in (1, 129, 512, 1024, 2048, 4096, 5000):
            for k in (1, 128, 1000, 1024, 2048, 4096, 14336):
                pol = module.heuristic_a8w8(m, n, k, False, True, sms)
                tiles = -(-n // 128) if pol["swap_ab"] else -(-m // 128) * -(-n // pol["tile_n"])
                if pol["split_k"] > 1:
                    assert tiles <= module._clusters(pol["split_k"], sms)
                    assert pol["split_k"] <= -(-k // 128)  # no CTA without a block


@pytest.mark.parametrize("group", [-3, 0, 1, 2, 3, 4, 1 << 20, 1 << 30, (1 << 31) - 1])
@pytest.mark.parametrize("m,n,kw", [(700, 520, dict(tile_n=128)), (520, 700, dict(tile_n=128, swap_ab=1)), (700, 1030, dict(tile_n=256, cta_group=2)), (1, 1 << 30, dict(tile_n=16))])
def test_a_group_of_tile_rows_is_no_larger_than_the_matrix(group, m, n, kw):
    # the kernel multiplies the group by the tiles in a row, in 32 bits; here its walk is taken over all tiles, or the first and last
    a = args8(m=m, n=n, ldo=n, ldb=256, **kw)
    a.policy.group_m = group
    pl = _lib.Plan()
    assert _lib.load().b200_gemm_a8w8_plan_query(C.byref(a), C.byref(pl)) == 0
    assert 0 <= pl.group_m <= pl.tiles_p and (pl.group_m > 0) == (group > 0)
    assert pl.group_m * pl.tiles_q < 1 << 31
    total = pl.tiles_p * pl.tiles_q
    if pl.group_m and total < 10000:
        seen = set()
        for tile in range(total):
            g, r = divmod(tile, pl.group_m * pl.tiles_q)
            rows = min(pl.tiles_p - g * pl.group_m, pl.group_m)
            seen.add((g * pl.group_m + r % rows, r // rows))
        assert seen == {(p, q) for p in range(pl.tiles_p) for q in range(pl.tiles_q)}


def test_quantizer_refuses_scales_and_sums_off_their_alignment():
    # fp32 stores to such addresses would fault; exponent tiles are bytes and start anywhere
    def quant(**kw):
        q = _lib.QuantizeArgs()
        base = dict(x=4096, rows=4, cols=64, ldx=64, in_dtype=2, out_dtype=4, mode=3, q_row=4096, ldq_row=64, s_row=4096, sr_row=1, sr_group=4,
                    q_col=4096, ldq_col=64, s_col=4096, sc_group=64, sc_col=1)
        for key, v in {**base, **kw}.items():
            setattr(q, key, v)
        return _lib.load().b200_gemm_quantize_a8(C.byref(q), None)
    for off in (1, 2, 3):
        assert quant(s_row=4096 + off) == -1 and quant(s_col=4096 + off) == -1 and quant(colsum=4096 + off, colsum_ld=64) == -1
        assert quant(colsum=4096 + off, colsum_ld=64, packed=1) == -1
        assert quant(mode=4, s_row=4096 + off) == -1 and quant(mode=2, s_col=4096 + off) == -1
