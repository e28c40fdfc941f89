"""Rotations and the 8-bit cache without a GPU: the plan of a rotation, and
the refusals that need no device (CPU only)."""
import ctypes as C

import numpy as np
import pytest
import torch

import picolm_b200 as pb
from tests.kv8_util import frequencies

GOOD = dict(n_layers=2, n_heads=8, n_kv_heads=2, head_dim=64, n_pages=10, n_seqs=3, max_pages=4, fmt=pb.PL_KV8_INT8)


@pytest.mark.parametrize("dim,kw", [
    (64, {}), (128, dict(base=500000.0)), (2, {}), (0, {}), (90, dict(scaling=pb.PL_ROPE_SCALE_LINEAR, factor=3.0)),
    (128, dict(scaling=pb.PL_ROPE_SCALE_LLAMA3, base=500000.0, factor=8.0, orig_len=8192, low=1.0, high=4.0)),
    (64, dict(scaling=pb.PL_ROPE_SCALE_YARN, base=10000.0, factor=4.0, orig_len=4096, low=1.0, high=32.0)),
    (128, dict(scaling=pb.PL_ROPE_SCALE_YARN, base=1e6, factor=40.0, orig_len=32768, low=1.0, high=32.0))])
def test_frequencies_of_a_rotation(dim, kw):
    r = pb.Rope(128, dim=dim, **kw).struct
    freq, gain = frequencies(dim, **kw)
    got = np.array(r.half_turns[:dim // 2]) * np.pi
    assert np.allclose(got, freq.numpy(), rtol=1e-14, atol=0)
    assert r.gain == pytest.approx(gain, rel=1e-15) and all(x == 0 for x in r.half_turns[dim // 2:])


@pytest.mark.parametrize("args,rc", [
    (dict(head_dim=60), pb.PL_EUNSUPPORTED), (dict(head_dim=264), pb.PL_EUNSUPPORTED),
    (dict(head_dim=64, dim=66), pb.PL_EARG), (dict(head_dim=64, dim=3), pb.PL_EARG),
    (dict(head_dim=64, rope_type=2), pb.PL_EARG), (dict(head_dim=64, base=0.0), pb.PL_EARG),
    (dict(head_dim=64, base=float("nan")), pb.PL_EARG), (dict(head_dim=64, scaling=4), pb.PL_EARG),
    (dict(head_dim=64, scaling=1, factor=0.5), pb.PL_EARG), (dict(head_dim=64, scaling=2, factor=2.0), pb.PL_EARG),
    (dict(head_dim=64, scaling=3, factor=2.0, orig_len=10, low=4.0, high=4.0), pb.PL_EARG)])
def test_rotations_that_are_refused(args, rc):
    with pytest.raises(pb.PlAttnError) as e:
        pb.Rope(**args)
    assert e.value.rc == rc


@pytest.mark.parametrize("change,rc", [
    ({}, pb.PL_OK), (dict(head_dim=96), pb.PL_EUNSUPPORTED), (dict(n_heads=18), pb.PL_EUNSUPPORTED),
    (dict(n_heads=9), pb.PL_EUNSUPPORTED), (dict(n_heads=14), pb.PL_OK), (dict(n_pages=0), pb.PL_EARG),
    (dict(n_seqs=-1), pb.PL_EARG), (dict(max_pages=2 ** 26), pb.PL_EARG), (dict(fmt=2), pb.PL_EARG),
    (dict(n_pages=2 ** 30), pb.PL_EUNSUPPORTED)])
def test_shapes_of_a_cache(change, rc):
    if rc == pb.PL_OK:
        assert pb.kv8_work_bytes(**{**GOOD, **change}) >= 256
        return
    with pytest.raises(pb.PlAttnError) as e:
        pb.kv8_work_bytes(**{**GOOD, **change})
    assert e.value.rc == rc


def test_calls_without_a_device_or_with_bad_pointers():
    """Every call checks its cache before it touches a device."""
    lib = pb.load()
    c = pb.Kv8Cache(**GOOD, codes=256, scales=256, table=256, lens=256, refs=256, work=256,
                    work_bytes=pb.kv8_work_bytes(**GOOD))
    p, P = c._p, 4096
    calls = {
        "resize": lambda x: lib.pl_kv8_resize_dev(x, 1, P, P, None),
        "fork": lambda x: lib.pl_kv8_fork_dev(x, 1, P, P, None),
        "compact": lambda x: lib.pl_kv8_compact_dev(x, None),
        "copy": lambda x: lib.pl_kv8_copy_dev(x, 1, P, P, None),
        "append": lambda x: lib.pl_kv8_append_dev(x, 0, 1, P, P, 1, 1, 0, P, 128, P, 128, None),
        "attend": lambda x: lib.pl_kv8_attend_dev(x, 0, 1, P, P, 1, 1, 0, P, 512, P, 512, None),
        "decode": lambda x: lib.pl_kv8_decode_dev(x, 0, 1, P, 0, P, 512, P, 128, P, 128, P, 512, None),
        "read": lambda x: lib.pl_kv8_read_dev(x, 0, 1, P, P, P, 1, 1, 0, P, 128, P, 128, None),
        "status": lambda x: lib.pl_kv8_status(x, None),
    }
    for name, call in calls.items():
        assert call(None) == pb.PL_EARG, name
        if not torch.cuda.is_available():
            assert call(p) == pb.PL_EDEVICE, name
        for field, value in (("codes", 0), ("codes", 128), ("work", 64), ("table", 2), ("work_bytes", 100),
                             ("head_dim", 32), ("format", 7)):
            old = getattr(c.struct, field)
            setattr(c.struct, field, value)
            assert call(p) in (pb.PL_EARG, pb.PL_EUNSUPPORTED), (name, field)
            setattr(c.struct, field, old)
    if torch.cuda.is_available():
        return
    with pytest.raises(pb.PlAttnError) as e:
        pb.Kv8Cache(**GOOD)
    assert e.value.rc == pb.PL_EDEVICE


def test_rope_rows_refusals_need_no_device():
    lib = pb.load()
    r = pb.Rope(64)
    P = 4096

    def call(dtype=0, n=1, pos=P, h=2, q=P, qs=128, qo=P, qos=128, rope=r._p):
        return lib.pl_rope_rows_dev(rope, dtype, n, pos, h, q, qs, qo, qos, 0, None, 0, None, 0, 0, None)

    assert call(n=0) == pb.PL_OK and call(h=0) == pb.PL_OK
    for bad in (dict(dtype=3), dict(n=-1), dict(pos=None), dict(h=-1), dict(q=None), dict(qs=127), dict(qo=None),
                dict(qos=1), dict(rope=None), dict(q=4097)):
        assert call(**bad) == pb.PL_EARG, bad
    r.struct.dim = 65
    assert call() == pb.PL_EARG


def test_struct_sizes_match_the_header(tmp_path):
    """ctypes and C agree on pl_rope and pl_kv8."""
    import os
    import shutil
    import subprocess
    if shutil.which("gcc") is None:
        pytest.skip("gcc not found")
    src = tmp_path / "size.c"
    src.write_text('#include <stdio.h>\n#include "pl_attn.h"\nint main(void) { printf("%zu %zu %zu\\n", '
                   "sizeof(pl_rope), sizeof(pl_kv8), offsetof(pl_kv8, codes)); return 0; }\n")
    subprocess.run(["gcc", "-std=c11", "-I", os.path.dirname(pb.HEADER), "-o", str(tmp_path / "size"), str(src)], check=True)
    got = subprocess.run([str(tmp_path / "size")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in got] == [C.sizeof(pb._RopeStruct), C.sizeof(pb._Kv8Struct), pb._Kv8Struct.codes.offset]


def test_layouts_that_do_not_exist_are_refused():
    r = pb.Rope(64)
    r.struct.type = 2
    P = 4096
    assert pb.load().pl_rope_rows_dev(r._p, 0, 1, P, 2, P, 128, P, 128, 0, None, 0, None, 0, 0, None) == pb.PL_EARG
    c = pb.Kv8Cache(**GOOD, rope=r, codes=256, scales=256, table=256, lens=256, refs=256, work=256,
                    work_bytes=pb.kv8_work_bytes(**GOOD))
    assert pb.load().pl_kv8_status(c._p, None) == pb.PL_EARG
