"""CPU tests of the paged cache's C boundary: struct layouts, sizes and the refusals that need no device."""
import ctypes
import shutil
import subprocess

import pytest

from rta_b200 import _build, _lib


@pytest.mark.parametrize("mirror,name", [(_lib.PagePoolC, "rta_page_pool"), (_lib.PageMapC, "rta_page_map")])
def test_struct_mirrors_have_the_c_layout(tmp_path, mirror, name):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    fields = [f[0] for f in mirror._fields_]
    src = tmp_path / "layout.c"
    src.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"rta.h\"\nint main(void) {\n"
                   f"  printf(\"%zu\\n\", sizeof({name}));\n"
                   + "".join(f"  printf(\"%zu\\n\", offsetof({name}, {f}));\n" for f in fields) + "  return 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run([cc, "-I", str(_build.INCLUDE), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(mirror)] + [getattr(mirror, f).offset for f in fields]


BASE = 1 << 20  # addresses that are only checked, never read


def pool(**kw):
    d = dict(k=BASE, v=BASE, format=1, layers=2, pages=8, page_size=16, kv_heads=2, head_dim=64, layer_stride=16384,
             page_stride=2048, head_stride=1024, position_stride=64)
    d.update(kw)
    return _lib.PagePoolC(*[d[f[0]] for f in _lib.PagePoolC._fields_])


def pmap(**kw):
    d = dict(refs=BASE, table=BASE + 4096, lengths=BASE + 8192, slots=4, width=8)
    d.update(kw)
    return _lib.PageMapC(*[d[f[0]] for f in _lib.PageMapC._fields_])


def calls(lib, p, m, ws=BASE, n=1 << 40, layer=0, slots=None, batch=1, q=BASE, fmt=1, heads=4, row=256, head=64,
          scale=0.1, out=BASE, starts=BASE, rows=1, other=None, ints=BASE, count=1):
    p, m = ctypes.byref(p), ctypes.byref(m)
    o = m if other is None else ctypes.byref(other)
    return {
        "decode": lib.rta_paged_decode(p, m, layer, slots, batch, q, fmt, heads, row, head, scale, 0, 0, out, None, ws,
                                       n, None),
        "prefill": lib.rta_paged_prefill(p, m, layer, slots, batch, starts, rows, q, fmt, heads, row, head, scale, 0,
                                         0, out, None, ws, n, None),
        "append": lib.rta_paged_append(p, m, layer, slots, batch, starts, rows, q, q, fmt, row, head, ws, n, None),
        "reserve": lib.rta_pages_reserve(p, m, o, slots, ints, count, ws, n, None),
        "fork": lib.rta_pages_fork(p, m, o, ints, ints, count, ws, n, None),
        "free": lib.rta_pages_free(p, m, o, ints, count, ws, n, None),
        "compact": lib.rta_pages_compact(p, m, o, None, ws, n, None),
        "copy": lib.rta_pages_copy(p, ints, ints, count, ws, n, None)}


ALL = {"decode", "prefill", "append", "reserve", "fork", "free", "compact", "copy"}
ATTEND = {"decode", "prefill"}
ROWS = ATTEND | {"append"}
BOOKS = {"reserve", "fork", "free", "compact"}


@pytest.mark.parametrize("refused,kw", [
    (ALL, {"p": pool(k=None)}), (ALL, {"p": pool(format=0)}), (ALL, {"p": pool(head_dim=96)}),
    (ALL, {"p": pool(page_size=0)}), (ALL, {"p": pool(page_size=65537)}), (ALL, {"p": pool(pages=0)}),
    (ALL, {"p": pool(position_stride=68)}), (ALL, {"p": pool(v=BASE + 8)}), (ALL, {"p": pool(kv_heads=0)}),
    (ALL - {"copy"}, {"m": pmap(table=None)}), (ALL - {"copy"}, {"m": pmap(width=1 << 27)}),
    (ALL - {"copy"}, {"m": pmap(slots=0)}), (ALL, {"ws": None}), (ALL, {"ws": BASE + 4}), (ALL, {"n": 1000}),
    (ROWS, {"layer": 2}), (ROWS, {"batch": 0}), (ROWS, {"batch": 5}), (ROWS, {"q": None}), (ROWS, {"q": BASE + 2}),
    (ROWS, {"row": 257}), (ROWS, {"fmt": 30}), ({"prefill"}, {"fmt": 0}), (ATTEND, {"heads": 3}),
    (ATTEND, {"heads": 258}), (ATTEND, {"out": None}), (ATTEND, {"scale": float("inf")}),
    ({"prefill", "append"}, {"starts": None}), ({"prefill"}, {"rows": 0}), ({"prefill"}, {"rows": 1 << 30}),
    (BOOKS, {"other": pmap(slots=3)}), (BOOKS, {"other": pmap(table=BASE + 12288)}),
    ({"reserve", "fork", "free", "copy"}, {"ints": None}), ({"reserve", "fork", "free", "copy"}, {"count": 0}),
    ({"reserve", "fork", "free"}, {"count": 5}), ({"reserve", "fork", "free", "copy"}, {"count": 9}),
], ids=lambda x: "" if isinstance(x, set) else ",".join(x))
def test_bad_arguments_are_refused(refused, kw):
    """Host-side checks answer RTA_E_ARG, with a text that names the call, before anything is launched."""
    if _gpu():
        pytest.skip("made-up addresses: calls that are not refused must not reach a device")
    lib = _lib.load()
    kw = {"p": pool(), "m": pmap(), **kw}
    for name, status in calls(lib, **kw).items():
        assert (status == _lib.RTA_E_ARG) == (name in refused), (name, status)


def _gpu():
    import torch
    return torch.cuda.is_available()


@pytest.mark.parametrize("slots", [None, BASE])
def test_a_batch_past_31_bits_is_refused(slots):
    """The kernels count sequences in 32 bits, some hundred at a time."""
    if _gpu():
        pytest.skip("made-up addresses: calls that are not refused must not reach a device")
    status = calls(_lib.load(), pool(), pmap(), slots=slots, batch=0xffffffff)
    assert {name for name in ROWS if status[name] == _lib.RTA_E_ARG} == ROWS


def test_refusals_name_the_call():
    lib = _lib.load()
    assert lib.rta_paged_decode(None, None, 0, None, 1, None, 1, 4, 0, 0, 1.0, 0, 0, None, None, None, 0, None) == 1
    assert lib.rta_last_error().startswith(b"rta_paged_decode: ")
    assert lib.rta_pages_compact(ctypes.byref(pool()), None, None, None, None, 0, None) == 1
    assert lib.rta_last_error().startswith(b"rta_pages_compact: ")


def test_workspace_bytes():
    lib = _lib.load()
    small = lib.rta_paged_workspace_bytes(ctypes.byref(pool()), ctypes.byref(pmap()))
    large = lib.rta_paged_workspace_bytes(ctypes.byref(pool(pages=1 << 26)), ctypes.byref(pmap()))
    assert 0 < small < large and large >= 16 << 26
    assert lib.rta_paged_workspace_bytes(ctypes.byref(pool(head_dim=1)), ctypes.byref(pmap())) == 0
