"""Operators on device tensors: what can be said without a GPU.  Struct layouts, the form of a tile, and the calls that are refused before anything
reaches a device."""
import ctypes as C
import os
import struct
import subprocess

import pytest

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EINVAL, ELIMIT = 1, 5


def test_tiles_and_look_ups(tmp_path):
    out = str(tmp_path / "pages4_main")
    subprocess.run(["g++", "-std=c++17", "-I" + os.path.join(ROOT, "linmt_b200", "csrc"), os.path.join(ROOT, "tests", "cpp", "pages4_main.cpp"), "-o", out], check=True)
    r = subprocess.run([out], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


PTR = 4096      # an aligned address that a refused call never follows

# Argument structs as C lays them out: (name, fields).  An entry is a format character with a default.
STRUCTS = {
    "linmt_beam_select_args": [("size", "I", 0), ("device", "i", 0), ("stream", "P", 0), ("logits", "P", PTR), ("stride_n", "q", 4000), ("stride_k", "q", 1000), ("scores", "P", PTR),
                               ("done", "P", 0), ("allowed", "P", 0), ("allowed_stride", "q", 0), ("out_tokens", "P", PTR), ("out_parents", "P", PTR), ("out_scores", "P", PTR), ("out_done", "P", PTR),
                               ("n", "i", 2), ("k", "i", 4), ("vocab", "i", 1000), ("eos", "i", 1), ("dtype", "i", 0), ("pad", "4x", None)],
    "linmt_plan_pages_args": [("size", "I", 0), ("device", "i", 0), ("stream", "P", 0), ("old_len", "P", 0), ("new_len", "P", PTR), ("table", "P", PTR), ("table_stride", "q", 4), ("free_pages", "P", PTR),
                              ("used", "P", PTR), ("out_used", "P", 2 * PTR), ("out_slots", "P", PTR), ("out_starts", "P", PTR), ("n", "i", 2), ("width", "i", 4), ("page", "i", 16), ("n_free", "i", 8), ("total", "q", 10)],
    "linmt_pages4_rows_args": [("size", "I", 0), ("device", "i", 0), ("stream", "P", 0), ("data", "P", PTR), ("stride_page", "q", 2304), ("stride_head", "q", 1152), ("n_pages", "i", 4), ("heads", "i", 2), ("page", "i", 16), ("dim", "i", 64),
                               ("slots", "P", PTR), ("k", "P", PTR), ("v", "P", PTR), ("k_stride_t", "q", 128), ("k_stride_h", "q", 64), ("v_stride_t", "q", 128), ("v_stride_h", "q", 64), ("t", "i", 3), ("dtype", "i", 1)],
    "linmt_attend_pages4_args": [("size", "I", 0), ("device", "i", 0), ("stream", "P", 0), ("data", "P", PTR), ("stride_page", "q", 2304), ("stride_head", "q", 1152), ("n_pages", "i", 4), ("heads_pool", "i", 2), ("page", "i", 16), ("dim", "i", 64),
                                 ("q", "P", PTR), ("q_stride_n", "q", 256), ("q_stride_g", "q", 128), ("q_stride_h", "q", 64), ("out", "P", PTR), ("out_stride_n", "q", 256), ("out_stride_g", "q", 128), ("out_stride_h", "q", 64),
                                 ("lse", "P", 0), ("table", "P", PTR), ("table_stride", "q", 4), ("len", "P", PTR), ("slope", "P", 0), ("centre", "P", 0), ("first", "P", 0), ("last", "P", 0), ("workspace", "P", 0), ("workspace_bytes", "q", 0),
                                 ("n", "i", 2), ("g", "i", 2), ("heads", "i", 2), ("width", "i", 4), ("dtype", "i", 1), ("scale", "f", 0.125), ("cap", "f", 0.0), ("pad", "4x", None)],
}


def _pack(name, **kw):
    fields = STRUCTS[name]
    fmt = struct.Struct("@" + "".join(f for _, f, _ in fields))
    kw.setdefault("size", fmt.size)
    values = [kw.get(n, d) for n, f, d in fields if d is not None]
    assert set(kw) <= {n for n, _, _ in fields}
    return fmt.pack(*values)


def test_struct_layouts(tmp_path):
    """Field by field as the C compiler lays the header's structs out."""
    rename = {("linmt_pages4_rows_args", n): "pages." + n for n in ("data", "stride_page", "stride_head", "n_pages", "heads", "page", "dim")}
    rename.update({("linmt_attend_pages4_args", n): "pages." + n for n in ("data", "stride_page", "stride_head", "n_pages", "page", "dim")})
    rename[("linmt_attend_pages4_args", "heads_pool")] = "pages.heads"
    lines, want = [], []
    for name, fields in STRUCTS.items():
        at = ""
        for n, f, d in fields:
            if d is not None:
                lines.append(f'printf("%zu\\n", offsetof({name}, {rename.get((name, n), n)}));')
                want.append(struct.calcsize("@" + at + f) - struct.calcsize(f))
            at += f
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(struct.calcsize("@" + at))
    src = tmp_path / "layout.c"
    src.write_text('#include "linmt_decoder.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    subprocess.run(["gcc", "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == want


def _refused(lib, fn, name, code, word, **kw):
    assert getattr(lib, fn)(_pack(name, **kw)) == code
    assert word in lib.linmt_op_error().decode(), lib.linmt_op_error()


@pytest.mark.parametrize("code,word,kw", [
    (EINVAL, "struct", dict(size=8)), (EINVAL, "missing", dict(logits=0)), (EINVAL, "missing", dict(out_tokens=0)), (EINVAL, "k = 0", dict(k=0)), (EINVAL, "n = -1", dict(n=-1)),
    (EINVAL, "vocab = 0", dict(vocab=0)), (EINVAL, "dtype = 3", dict(dtype=3)), (EINVAL, "eos", dict(eos=1000)), (EINVAL, "eos", dict(eos=-1)), (EINVAL, "aligned", dict(logits=PTR + 2)),
    (EINVAL, "aligned", dict(logits=PTR + 1, dtype=1)), (EINVAL, "aligned", dict(allowed=PTR + 1)), (ELIMIT, "k = 33", dict(k=33)), (ELIMIT, "2^31", dict(k=32, vocab=1 << 26))])
def test_beam_select_refuses(cuda_lib, code, word, kw):
    _refused(cuda_lib, "linmt_beam_select", "linmt_beam_select_args", code, word, **kw)


@pytest.mark.parametrize("code,word,kw", [
    (EINVAL, "struct", dict(size=8)), (EINVAL, "page = 0", dict(page=0)), (EINVAL, "total = -1", dict(total=-1)), (EINVAL, "read and written", dict(out_used=PTR)), (EINVAL, "missing", dict(new_len=0)),
    (EINVAL, "missing", dict(table=0)), (EINVAL, "aligned", dict(out_slots=PTR + 4)), (ELIMIT, "16384", dict(n=16385)), (ELIMIT, "2^31", dict(n=16384, width=1 << 18)), (ELIMIT, "2^31", dict(total=1 << 31))])
def test_plan_pages_refuses(cuda_lib, code, word, kw):
    _refused(cuda_lib, "linmt_plan_pages", "linmt_plan_pages_args", code, word, **kw)


@pytest.mark.parametrize("fn", ["linmt_write_pages4", "linmt_read_pages4"])
@pytest.mark.parametrize("code,word,kw", [
    (EINVAL, "struct", dict(size=8)), (EINVAL, "pool", dict(page=24)), (EINVAL, "pool", dict(page=0)), (EINVAL, "pool", dict(n_pages=0)), (EINVAL, "pool", dict(data=0)), (ELIMIT, "dim = 96", dict(dim=96)),
    (EINVAL, "16 bytes", dict(data=PTR + 8)), (EINVAL, "16 bytes", dict(stride_head=1160)), (EINVAL, "missing", dict(v=0)), (EINVAL, "16 bytes", dict(k=PTR + 8)), (EINVAL, "16 bytes", dict(v_stride_h=68)),
    (EINVAL, "dtype", dict(dtype=9)), (EINVAL, "t = -1", dict(t=-1))])
def test_rows_refuse(cuda_lib, fn, code, word, kw):
    _refused(cuda_lib, fn, "linmt_pages4_rows_args", code, word, **kw)


@pytest.mark.parametrize("code,word,kw", [
    (EINVAL, "struct", dict(size=8)), (EINVAL, "multiple of the pool", dict(heads=3)), (EINVAL, "heads = 0", dict(heads=0)), (EINVAL, "missing", dict(q=0)), (EINVAL, "missing", dict(len=0)),
    (EINVAL, "slope goes with", dict(slope=PTR)), (EINVAL, "first with last", dict(last=PTR)), (EINVAL, "finite", dict(scale=float("nan"))), (EINVAL, "finite", dict(cap=float("inf"))), (EINVAL, "finite", dict(cap=-1.0)), (EINVAL, "too small", dict(cap=1e-30)),
    (EINVAL, "aligned", dict(q=PTR + 1)), (ELIMIT, "dim = 32", dict(dim=32)), (EINVAL, "workspace", dict(width=4096)), (EINVAL, "workspace", dict(width=4096, workspace=PTR, workspace_bytes=64)), (ELIMIT, "too many", dict(n=1 << 24))])
def test_attend_refuses(cuda_lib, code, word, kw):
    _refused(cuda_lib, "linmt_attend_pages4", "linmt_attend_pages4_args", code, word, **kw)


def test_attend_workspace(cuda_lib):
    size = lambda **kw: cuda_lib.linmt_attend_pages4_workspace(_pack("linmt_attend_pages4_args", **kw))
    assert size(width=16) == 0 and size(n=0, width=4096) == 0 and size(heads=3) == -1     # sentences of up to 256 positions are not cut
    part = 16 * 66 * 4 + 8                                     # 16 rows: 64 sums, a maximum and a weight; two of them and 16 bytes for each CTA
    assert size(width=4096) == 592 * 2 * part and size(width=4096, n=4000) == 592 * 2 * part
    assert size(width=32) == 2 * 2 * 4 * 2 * part               # 2 sentences, 2 heads, 16 pairs of tiles that count as 28 units, in parts of 8


def test_nothing_to_do_reaches_no_device(cuda_lib):
    assert cuda_lib.linmt_beam_select(_pack("linmt_beam_select_args", n=0)) == 0
    assert cuda_lib.linmt_write_pages4(_pack("linmt_pages4_rows_args", t=0)) == 0
    assert cuda_lib.linmt_attend_pages4(_pack("linmt_attend_pages4_args", n=0)) == 0
    assert cuda_lib.linmt_attend_pages4(_pack("linmt_attend_pages4_args", g=0)) == 0


def test_beam_reorder_refuses(cuda_lib):
    def args(n=2, k=4, n_states=1, parents=PTR, size=None, **st):
        s = dict(src=PTR, dst=PTR, sl=0, sn=64, sk=16, dl=0, dn=64, dk=16, row=16, layers=1)
        s.update(st)
        state = struct.pack("@PPqqqqqqqq", *s.values())
        return struct.pack("@IiPPiiii", 1320 if size is None else size, 0, 0, parents, n, k, n_states, 0) + state.ljust(16 * 80, b"\0")

    for code, word, kw in [(EINVAL, "struct", dict(size=8)), (EINVAL, "parents", dict(parents=0)), (EINVAL, "17 states", dict(n_states=17)), (ELIMIT, "k = 33", dict(k=33)), (EINVAL, "missing", dict(dst=0)),
                           (EINVAL, "two sets of strides", dict(dk=32)), (EINVAL, "layers", dict(layers=-1)), (ELIMIT, "blocks", dict(row=1 << 50))]:
        assert cuda_lib.linmt_beam_reorder(args(**kw)) == code, kw
        assert word in cuda_lib.linmt_op_error().decode(), kw
    assert cuda_lib.linmt_beam_reorder(args(n=0)) == 0 and cuda_lib.linmt_beam_reorder(args(n_states=0)) == 0 and cuda_lib.linmt_beam_reorder(args(row=0)) == 0


def test_tensors_of_the_host_are_refused(cuda_lib):
    from linmt_b200 import device_ops as ops
    x = torch.zeros
    with pytest.raises(ValueError, match="CUDA"):
        ops.beam_select(x(1, 2, 10), x(1, 2))
    with pytest.raises(ValueError, match="CUDA"):
        ops.beam_reorder([x(1, 2, 10)], x(1, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        ops.plan_pages(None, x(3, dtype=torch.int32), x(3, 4, dtype=torch.int32), x(9, dtype=torch.int32), x(1, dtype=torch.int32), page=16, total=4)
    pool = x(2, 1, 1, 18 * 64, dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA"):
        ops.write_pages4(pool, x(3, dtype=torch.int64), x(3, 1, 64), x(3, 1, 64))
    with pytest.raises(ValueError, match="CUDA"):
        ops.read_pages4(pool, x(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        ops.attend_pages4(x(1, 1, 1, 64), pool, x(1, 1, dtype=torch.int32), x(1, dtype=torch.int32))
