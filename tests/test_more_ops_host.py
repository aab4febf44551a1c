"""Memories in 8 bits, page plans, copies and scores: what can be said without a GPU.  Struct layouts, the form of a block, and the calls that are refused before anything reaches a device."""
import os
import struct
import subprocess

import pytest

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EINVAL, ELIMIT = 1, 5
PTR = 4096      # an aligned address that a refused call never follows


def test_blocks_and_look_ups(tmp_path):
    out = str(tmp_path / "pages8_main")
    subprocess.run(["g++", "-std=c++17", "-I" + os.path.join(ROOT, "linmt_b200", "csrc"), os.path.join(ROOT, "tests", "cpp", "pages8_main.cpp"), "-o", out], check=True)
    r = subprocess.run([out], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


_HEAD = [("size", "I", 0), ("device", "i", 0), ("stream", "P", 0)]
_POOL = [("data", "P", PTR), ("stride_page", "q", 2 * 2064), ("stride_head", "q", 2064), ("n_pages", "i", 4), ("heads_pool", "i", 2), ("page", "i", 16), ("dim", "i", 64)]

# Argument structs as C lays them out: (name, format, default).
STRUCTS = {
    "linmt_pages8_rows_args": _HEAD + _POOL + [("slots", "P", PTR), ("k", "P", PTR), ("v", "P", PTR), ("k_stride_t", "q", 128), ("k_stride_h", "q", 64), ("v_stride_t", "q", 128), ("v_stride_h", "q", 64), ("t", "i", 3), ("dtype", "i", 1)],
    "linmt_attend_pages8_args": _HEAD + _POOL + [("q", "P", PTR), ("q_stride_n", "q", 256), ("q_stride_g", "q", 128), ("q_stride_h", "q", 64), ("out", "P", PTR), ("out_stride_n", "q", 256), ("out_stride_g", "q", 128), ("out_stride_h", "q", 64),
                                                 ("lse", "P", 0), ("table", "P", PTR), ("table_stride", "q", 4), ("len", "P", PTR), ("slope", "P", 0), ("centre", "P", 0), ("first", "P", 0), ("last", "P", 0), ("workspace", "P", 0), ("workspace_bytes", "q", 0),
                                                 ("n", "i", 2), ("g", "i", 2), ("heads", "i", 2), ("width", "i", 4), ("dtype", "i", 1), ("sinks", "i", 0), ("scale", "f", 0.125), ("cap", "f", 0.0)],
    "linmt_fork_pages_args": _HEAD + [("table", "P", PTR), ("table_stride", "q", 4), ("len", "P", PTR), ("parents", "P", 0), ("done", "P", 0), ("shares", "P", PTR), ("free_pages", "P", PTR), ("used", "P", PTR), ("out_table", "P", PTR), ("out_table_stride", "q", 4),
                                      ("out_len", "P", PTR), ("out_shares", "P", PTR), ("out_free", "P", PTR), ("out_used", "P", PTR), ("out_src", "P", PTR), ("out_dst", "P", PTR), ("n", "i", 2), ("k", "i", 3), ("width", "i", 4), ("page", "i", 16), ("n_pages", "i", 30), ("n_free", "i", 30)],
    "linmt_compact_pages_args": _HEAD + [("table", "P", PTR), ("table_stride", "q", 4), ("len", "P", PTR), ("shares", "P", PTR), ("out_table", "P", PTR), ("out_table_stride", "q", 4), ("out_shares", "P", PTR), ("out_free", "P", PTR), ("out_used", "P", PTR),
                                         ("out_src", "P", PTR), ("out_dst", "P", PTR), ("workspace", "P", PTR), ("rows", "i", 6), ("width", "i", 4), ("page", "i", 16), ("n_pages", "i", 30)],
    "linmt_score_tokens_args": _HEAD + [("logits", "P", PTR), ("stride_n", "q", 4000), ("stride_t", "q", 1000), ("tokens", "P", PTR), ("allowed", "P", 0), ("allowed_stride", "q", 0), ("out_logprob", "P", PTR), ("out_entropy", "P", PTR), ("out_top_tokens", "P", 0),
                                        ("out_top_logprobs", "P", 0), ("n", "i", 2), ("t", "i", 4), ("vocab", "i", 1000), ("top", "i", 0), ("dtype", "i", 0), ("reserved", "i", 0)],
}


def _pack(name, **kw):
    fields = STRUCTS[name]
    fmt = struct.Struct("@" + "".join(f for _, f, _ in fields))
    kw.setdefault("size", fmt.size)
    assert set(kw) <= {n for n, _, _ in fields}
    return fmt.pack(*[kw.get(n, d) for n, _, d in fields])


def test_struct_layouts(tmp_path):
    """Field by field as the C compiler lays the header's structs out."""
    lines, want = [], []
    for name, fields in STRUCTS.items():
        at = ""
        for n, f, _ in fields:
            in_pool = n in {x for x, _, _ in _POOL} and "pages8" in name
            lines.append(f'printf("%zu\\n", offsetof({name}, {"pages." + n.replace("heads_pool", "heads") if in_pool else n}));')
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


@pytest.mark.parametrize("fn", ["linmt_write_pages8", "linmt_read_pages8"])
@pytest.mark.parametrize("code,word,kw", [
    (EINVAL, "struct", dict(size=8)), (EINVAL, "pool", dict(page=24)), (EINVAL, "pool", dict(page=0)), (EINVAL, "pool", dict(n_pages=0)), (EINVAL, "pool", dict(data=0)), (ELIMIT, "dim = 96", dict(dim=96)),
    (EINVAL, "16 bytes", dict(data=PTR + 8)), (EINVAL, "16 bytes", dict(stride_head=2072)), (EINVAL, "missing", dict(v=0)), (EINVAL, "16 bytes", dict(k=PTR + 8)), (EINVAL, "16 bytes", dict(v_stride_h=68)),
    (EINVAL, "dtype", dict(dtype=9)), (EINVAL, "t = -1", dict(t=-1)), (ELIMIT, "65536 heads", dict(heads_pool=65536))])
def test_rows_refuse(cuda_lib, fn, code, word, kw):
    _refused(cuda_lib, fn, "linmt_pages8_rows_args", code, word, **kw)


@pytest.mark.parametrize("code,word,kw", [
    (EINVAL, "struct", dict(size=8)), (EINVAL, "multiple of the pool", dict(heads=3)), (EINVAL, "heads = 0", dict(heads=0)), (EINVAL, "missing", dict(q=0)), (EINVAL, "missing", dict(len=0)), (EINVAL, "sinks = -1", dict(sinks=-1)),
    (EINVAL, "slope goes with", dict(slope=PTR)), (EINVAL, "first with last", dict(last=PTR)), (EINVAL, "finite", dict(scale=float("nan"))), (EINVAL, "finite", dict(cap=float("inf"))), (EINVAL, "finite", dict(cap=-1.0)), (EINVAL, "too small", dict(cap=1e-30)),
    (EINVAL, "aligned", dict(q=PTR + 1)), (ELIMIT, "dim = 32", dict(dim=32)), (EINVAL, "workspace", dict(width=4096)), (EINVAL, "workspace", dict(width=4096, workspace=PTR, workspace_bytes=64)), (EINVAL, "workspace", dict(width=4096, workspace=PTR + 4, workspace_bytes=1 << 30)),
    (ELIMIT, "too many", dict(n=1 << 24)), (ELIMIT, "too many", dict(n=1 << 14, width=1 << 20))])
def test_attend_refuses(cuda_lib, code, word, kw):
    _refused(cuda_lib, "linmt_attend_pages8", "linmt_attend_pages8_args", code, word, **kw)


def test_attend_workspace(cuda_lib):
    size = lambda **kw: cuda_lib.linmt_attend_pages8_workspace(_pack("linmt_attend_pages8_args", **kw))
    assert size(width=24) == 0 and size(n=0, width=4096) == 0 and size(heads=3) == -1     # sentences of up to 384 positions are not cut
    part = lambda rows: 2 * rows * 66 * 4 + 16                  # of each CTA two parts of 64 sums, an exponent and a weight for each row, and 16 bytes
    assert size(width=4096) == 2 * 2 * 86 * part(4) and size(width=16384) == 148 * 3 * part(4) and size(width=4096, g=5) == 148 * 2 * part(8) and size(width=4096, g=20) == 148 * 2 * part(16)
    assert size(width=32) == 2 * 2 * 2 * part(4)                # 2 sentences, 2 heads, 4 products that count as 7 units, in parts of 6


@pytest.mark.parametrize("code,word,kw", [
    (EINVAL, "struct", dict(size=8)), (EINVAL, "page = 0", dict(page=0)), (EINVAL, "n = -1", dict(n=-1)), (EINVAL, "missing", dict(len=0)), (EINVAL, "missing", dict(used=0)), (EINVAL, "missing", dict(out_dst=0)), (EINVAL, "missing", dict(out_table=0)),
    (EINVAL, "missing", dict(shares=0)), (EINVAL, "missing", dict(out_free=0)), (EINVAL, "aligned", dict(table=PTR + 2)), (EINVAL, "aligned", dict(parents=PTR + 1)), (ELIMIT, "16384", dict(n=4096, k=5)), (ELIMIT, "2^31", dict(n=1024, k=16, width=1 << 20))])
def test_fork_refuses(cuda_lib, code, word, kw):
    _refused(cuda_lib, "linmt_fork_pages", "linmt_fork_pages_args", code, word, **kw)


@pytest.mark.parametrize("code,word,kw", [
    (EINVAL, "struct", dict(size=8)), (EINVAL, "page = 0", dict(page=0)), (EINVAL, "rows = -1", dict(rows=-1)), (EINVAL, "missing", dict(len=0)), (EINVAL, "missing", dict(workspace=0)), (EINVAL, "missing", dict(out_src=0)), (EINVAL, "missing", dict(out_used=0)),
    (EINVAL, "aligned", dict(out_shares=PTR + 2)), (ELIMIT, "2^31", dict(rows=1 << 20, width=1 << 12))])
def test_compact_refuses(cuda_lib, code, word, kw):
    _refused(cuda_lib, "linmt_compact_pages", "linmt_compact_pages_args", code, word, **kw)


@pytest.mark.parametrize("code,word,kw", [
    (EINVAL, "struct", dict(size=8)), (EINVAL, "vocab = 0", dict(vocab=0)), (EINVAL, "top = -1", dict(top=-1)), (EINVAL, "dtype = 3", dict(dtype=3)), (EINVAL, "missing", dict(logits=0)), (EINVAL, "missing", dict(tokens=0)), (EINVAL, "missing", dict(top=3)),
    (EINVAL, "aligned", dict(logits=PTR + 2)), (EINVAL, "aligned", dict(logits=PTR + 1, dtype=1)), (EINVAL, "aligned", dict(allowed=PTR + 2)), (ELIMIT, "top = 33", dict(top=33)), (ELIMIT, "2^31", dict(n=1 << 16, t=1 << 16)), (ELIMIT, "2^31", dict(vocab=2 ** 31 - 1))])
def test_score_refuses(cuda_lib, code, word, kw):
    _refused(cuda_lib, "linmt_score_tokens", "linmt_score_tokens_args", code, word, **kw)


def test_copy_refuses(cuda_lib):
    def args(n=3, n_pages=5, n_pools=1, src=PTR, size=None, data=PTR, stride=64, page=64):
        head = struct.pack("@IiPPPiiii", 48 + 16 * 24 if size is None else size, 0, 0, src, PTR, n, n_pages, n_pools, 0)
        return head + (struct.pack("@Pqq", data, stride, page) * min(max(n_pools, 0), 16)).ljust(16 * 24, b"\0")

    for code, word, kw in [(EINVAL, "struct", dict(size=8)), (EINVAL, "17 pools", dict(n_pools=17)), (EINVAL, "n = -1", dict(n=-1)), (EINVAL, "missing", dict(src=0)), (EINVAL, "aligned", dict(src=PTR + 2)), (EINVAL, "pool 0", dict(data=0)),
                           (EINVAL, "pool 0", dict(page=-1)), (EINVAL, "overlap", dict(stride=32)), (ELIMIT, "too large", dict(stride=1 << 50, page=1 << 50))]:
        assert cuda_lib.linmt_copy_pages(args(**kw)) == code, kw
        assert word in cuda_lib.linmt_op_error().decode(), kw
    assert cuda_lib.linmt_copy_pages(args(n=0)) == 0 and cuda_lib.linmt_copy_pages(args(n_pools=0)) == 0 and cuda_lib.linmt_copy_pages(args(page=0)) == 0


def test_nothing_to_do_reaches_no_device(cuda_lib):
    assert cuda_lib.linmt_write_pages8(_pack("linmt_pages8_rows_args", t=0)) == 0
    assert cuda_lib.linmt_attend_pages8(_pack("linmt_attend_pages8_args", n=0)) == 0
    assert cuda_lib.linmt_attend_pages8(_pack("linmt_attend_pages8_args", g=0)) == 0
    assert cuda_lib.linmt_score_tokens(_pack("linmt_score_tokens_args", n=0)) == 0
    assert cuda_lib.linmt_score_tokens(_pack("linmt_score_tokens_args", t=0)) == 0


def test_tensors_of_the_host_are_refused(cuda_lib):
    from linmt_b200 import device_ops as ops
    x = torch.zeros
    i = lambda *s: torch.zeros(s, dtype=torch.int32)
    pool = x(2, 1, 1, 32 * 64 + 16, dtype=torch.uint8)
    for call in (lambda: ops.write_pages8(pool, x(3, dtype=torch.int64), x(3, 1, 64), x(3, 1, 64)), lambda: ops.read_pages8(pool, x(3, dtype=torch.int64)), lambda: ops.attend_pages8(x(1, 1, 1, 64), pool, i(1, 1), i(1)),
                 lambda: ops.fork_pages(i(1, 2, 3), i(1, 2), i(1, 2), i(9), i(9), i(1), page=16), lambda: ops.free_pages(i(2, 3), i(2), x(2, dtype=torch.bool), i(9), i(9), i(1), page=16),
                 lambda: ops.compact_pages(i(2, 3), i(2), i(9), page=16), lambda: ops.copy_pages([pool], i(2), i(2)), lambda: ops.score_tokens(x(1, 2, 10), i(1, 2))):
        with pytest.raises(ValueError, match="CUDA"):
            call()
