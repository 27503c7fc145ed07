"""CPU tests of the paged cache's boundary: the header's functions are exported and bound, the argument structures have the
C layout, and entry points and Python calls refuse what they cannot run before anything is launched."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "sisa_hip_cache.h")


@pytest.fixture(scope="module")
def lib():
    from sisa_amd.kernels import _lib
    if not os.path.exists(_lib.LIB_PATH):
        from sisa_amd import build
        build.build()
    return _lib.load()


def test_header_functions_are_exported(lib):
    from sisa_amd.kernels import _lib
    declared = set(re.findall(r"^(?:int|int64_t)\s+(sisa_\w+)\(", open(HEADER).read(), re.M))
    assert declared == set(_lib.CACHE_SIGNATURES) and len(declared) == 8
    assert all(hasattr(lib, name) for name in declared)


def test_struct_layout_matches_c(tmp_path):
    from sisa_amd.kernels import _lib
    pairs = {"PagePoolArgs": "sisa_page_pool", "PagedWriteArgs": "sisa_paged_write_args",
             "PagedDecodeArgs": "sisa_paged_decode_args", "AttnWeightsArgs": "sisa_attn_weights_args",
             "CacheEvictArgs": "sisa_cache_evict_args", "StepPagedArgs": "sisa_step_paged_args"}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "sisa_hip_cache.h"', "int main(void) {"]
    expect = []
    for py, c in pairs.items():
        cls = getattr(_lib, py)
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        expect.append(ctypes.sizeof(cls))
        for name, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({c}, {name.rstrip("_")}));')
            expect.append(getattr(cls, name).offset)
    lines += ["return 0;", "}"]
    (tmp_path / "layout.c").write_text("\n".join(lines))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(tmp_path / "layout.c"), "-o", str(exe)],
                   check=True)
    assert [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()] == expect


def _pool(lib, **kw):
    from sisa_amd.kernels import _lib
    row, gate = _lib.View(4096, 2 * 16 * 64, 16 * 64, 64), _lib.View(4096, 32, 16, 1)
    p = dict(pages=2, heads=2, page_size=16, dtype=_lib.BF16, k=row, v=row, b=row, g=gate, f=gate) | kw
    return _lib.PagePoolArgs(*p.values())


def _refused(lib, name, args, word):
    assert getattr(lib, name)(ctypes.byref(args), None) == 1, word
    message = lib.sisa_last_error().decode()
    assert message.startswith(name) and word in message, message


def test_entry_points_refuse_bad_arguments(lib):
    from sisa_amd.kernels import _lib
    none, row, gate = _lib.View(None, 0, 0, 0), _lib.View(4096, 1024, 64, 64), _lib.View(4096, 32, 16, 1)
    crooked = _lib.View(4104, 1024, 64, 64)
    for name in ("sisa_paged_write", "sisa_paged_decode", "sisa_attn_weights", "sisa_cache_evict"):
        assert getattr(lib, name)(None, None) == 1 and lib.sisa_last_error().decode().startswith(name)

    def write(B=1, M=1, W=1, pool=None, table=4096, start=4096, k=row, f=gate):
        return _lib.PagedWriteArgs(B, M, W, 0, pool or _pool(lib), table, W, start, None, k, row, row, gate, f)
    for args, word in ((write(pool=_pool(lib, page_size=24)), "power of two"), (write(pool=_pool(lib, page_size=8)), "at least 16"),
                       (write(pool=_pool(lib, pages=0)), "pages and heads"), (write(pool=_pool(lib, dtype=3)), "dtype"),
                       (write(pool=_pool(lib, v=crooked)), "aligned"), (write(pool=_pool(lib, g=none)), "no g"),
                       (write(W=0), "bad shape"), (write(table=None), "table"), (write(k=crooked), "aligned"),
                       (write(f=none), "f where the pool has one")):
        _refused(lib, "sisa_paged_write", args, word)
    assert lib.sisa_paged_write(ctypes.byref(write(M=0)), None) == 0

    def decode(B=1, M=1, W=1, max_len=16, q=row, fq=gate, w_in=none, w_out=none, out=4096, ws=4096):
        return _lib.PagedDecodeArgs(B, M, W, max_len, _pool(lib), 4096, W, 4096, q, row, gate, fq, 4096, 1, w_in, w_out, out, ws)
    for args, word in ((decode(max_len=17), "max_len"), (decode(max_len=0), "max_len"), (decode(M=0), "M=0"),
                       (decode(q=crooked), "aligned"), (decode(fq=none), "fq"), (decode(w_in=gate), "together"),
                       (decode(out=None), "null"), (decode(W=100, max_len=1600, ws=None), "null workspace"),
                       (decode(W=100, max_len=1600, ws=4104), "aligned")):
        _refused(lib, "sisa_paged_decode", args, word)
    assert lib.sisa_paged_decode(ctypes.byref(decode(B=0)), None) == 0

    def weights(B=1, H=1, L=8, window=0, dtype=_lib.BF16, q=row, g=gate, out=4096):
        return _lib.AttnWeightsArgs(B, H, L, window, dtype, 0, q, row, row, row, g, none, 4096, 1, None, out, 4096)
    for args, word in ((weights(L=-1), "bad shape"), (weights(window=-1), "window=-1"), (weights(dtype=3), "dtype"),
                       (weights(q=crooked), "aligned"), (weights(g=none), "null"), (weights(out=None), "null")):
        _refused(lib, "sisa_attn_weights", args, word)
    assert lib.sisa_attn_weights(ctypes.byref(weights(L=0)), None) == 0

    def evict(B=1, keep=4, recent=2, max_len=16, to=None, w=gate, positions=4096):
        return _lib.CacheEvictArgs(B, 1, 1, max_len, keep, recent, _pool(lib), to or _pool(lib), 4096, 1, 4096, 1, 4096, w, 4096,
                                   4096, positions)
    for args, word in ((evict(recent=0), "recent"), (evict(recent=5), "recent"), (evict(max_len=17), "max_len"),
                       (evict(to=_pool(lib, heads=3)), "agree"), (evict(to=_pool(lib, dtype=2)), "agree"),
                       (evict(to=_pool(lib, f=none)), "agree"), (evict(w=none), "null"), (evict(positions=None), "null")):
        _refused(lib, "sisa_cache_evict", args, word)
    assert lib.sisa_cache_evict(ctypes.byref(evict(B=0)), None) == 0


def test_step_refuses_bad_arguments(lib):
    from sisa_amd.kernels import _lib
    assert lib.sisa_step_paged(None, None) == 1 and lib.sisa_last_error().decode().startswith("sisa_step_paged")

    def step(B=1, H=2, D=128, dtype=_lib.BF16, W=1, max_len=16, w_q=4096, pool=None, g_last=4096, ws=4096):
        return _lib.StepPagedArgs(B, H, D, 256, dtype, W, max_len, 0, 1e-6, 1e-6, 4096, D, None, 4096, w_q, *[4096] * 15,
                                  pool or _pool(lib), 4096, W, 4096, 4096, g_last, 4096, 4096, _lib.View(None, 0, 0, 0), 4096,
                                  4096, ws)
    none = _lib.View(None, 0, 0, 0)
    for args, word in ((step(B=0), "B must be"), (step(B=65), "B must be"), (step(D=192), "B must be"),
                       (step(dtype=_lib.F32), "bf16 or fp16"), (step(w_q=None), "given"), (step(w_q=4098), "aligned"),
                       (step(ws=4112), "256-byte"), (step(pool=_pool(lib, dtype=_lib.F16)), "heads and dtype"),
                       (step(pool=_pool(lib, heads=3)), "heads and dtype"), (step(pool=_pool(lib, f=none)), "and f"),
                       (step(pool=_pool(lib, page_size=20)), "power of two"), (step(max_len=17), "max_len"),
                       (step(g_last=None), "null")):
        _refused(lib, "sisa_step_paged", args, word)
    assert lib.sisa_step_paged_workspace_bytes(0, 2, 128, 256, 16, _lib.BF16, 0) == 0
    assert lib.sisa_step_paged_workspace_bytes(1, 2, 128, 256, 9000, _lib.BF16, 1) > \
        lib.sisa_step_paged_workspace_bytes(1, 2, 128, 256, 9000, _lib.BF16, 0) > 0


def test_workspaces(lib):
    from sisa_amd.kernels import _lib
    size = lib.sisa_paged_decode_workspace_bytes
    assert size(0, 1, 1, 1, _lib.BF16, 0) == 0
    one = size(2, 3, 1, 5000, _lib.BF16, 0)
    assert one > 0 and size(2, 3, 1, 5000, _lib.BF16, 1) == one + 2 * 3 * 5000 * 4
    # a cache that one workgroup takes whole needs none, but for the tracked weights of several rows
    assert size(2, 3, 1, 1024, _lib.BF16, 1) == size(2, 3, 4, 512, _lib.F32, 0) == 0
    assert size(2, 3, 2, 1024, _lib.BF16, 1) > 0 and size(2, 3, 1, 513, _lib.F32, 0) > 0
    assert lib.sisa_attn_weights_workspace_bytes(2, 3, 100, 0) >= 2 * 3 * 100 * 4
    assert lib.sisa_attn_weights_workspace_bytes(2, 3, 0, 0) == 0


def test_python_calls_refuse_tensors_off_the_gpu(lib):
    from sisa_amd.kernels import PagePool, sisa_attention_weights_hip
    z = torch.zeros
    with pytest.raises(ValueError, match="power of two"):
        PagePool(z(1, 1, 24, 64), z(1, 1, 24, 64), z(1, 1, 24, 32), z(1, 1, 24))
    with pytest.raises(ValueError, match="k and v"):
        PagePool(z(1, 1, 16, 32), z(1, 1, 16, 32), z(1, 1, 16, 32), z(1, 1, 16))
    with pytest.raises(TypeError, match="share"):
        PagePool(z(1, 1, 16, 64), z(1, 1, 16, 64).half(), z(1, 1, 16, 32), z(1, 1, 16))
    with pytest.raises(ValueError, match="GPU"):
        PagePool(z(1, 1, 16, 64), z(1, 1, 16, 64), z(1, 1, 16, 32), z(1, 1, 16))
    x = [z(1, 1, 4, 64), z(1, 1, 4, 64), z(1, 1, 4, 32), z(1, 1, 4, 32), z(1, 1, 4), z(1)]
    with pytest.raises(ValueError, match="GPU"):
        sisa_attention_weights_hip(*x)
    with pytest.raises(ValueError, match="c and b"):
        sisa_attention_weights_hip(x[0], x[1], x[2][:, :, :3], *x[3:])
    with pytest.raises(TypeError, match="share"):
        sisa_attention_weights_hip(x[0].half(), *x[1:])
    with pytest.raises(RuntimeError, match="inference"):
        sisa_attention_weights_hip(x[0].requires_grad_(True), *x[1:])


def test_entry_points_refuse_more_than_a_launch_takes(lib):
    """The threads of a launch are counted in 32 bits."""
    from sisa_amd.kernels import _lib
    none, row, gate = _lib.View(None, 0, 0, 0), _lib.View(4096, 1024, 64, 64), _lib.View(4096, 32, 16, 1)
    for B, M, W, w in ((1 << 14, 128, 100, none), (1 << 23, 1, 1, none), (1 << 22, 1, 32, gate)):
        args = _lib.PagedDecodeArgs(B, M, W, 16 * W, _pool(lib), 4096, W, 4096, row, row, gate, gate, 4096, 1, w, w, 4096, 4096)
        _refused(lib, "sisa_paged_decode", args, "too large")
    for B, H, L, window in ((1 << 14, 1 << 6, 2048, 0), (1, 1, 1 << 30, 300), (1 << 10, 1 << 10, 4096, 1)):
        args = _lib.AttnWeightsArgs(B, H, L, window, _lib.BF16, 0, row, row, row, row, gate, none, 4096, 1, None, 4096, 4096)
        _refused(lib, "sisa_attn_weights", args, "too large")
    args = _lib.CacheEvictArgs(1 << 21, 1, 1, 16, 4, 2, _pool(lib), _pool(lib), 4096, 1, 4096, 1, 4096, gate, 4096, 4096, 4096)
    _refused(lib, "sisa_cache_evict", args, "2^22")


@pytest.mark.parametrize("tracked", [False, True])
@pytest.mark.parametrize("max_len", [1 << 22, 1 << 24, 1 << 30])
def test_step_refuses_more_than_a_launch_takes(lib, max_len, tracked):
    """Chunks of 256 positions of 64 rows of 16 heads: 2^32 threads and more."""
    from sisa_amd.kernels import _lib
    weights = _lib.View(4096, 1 << 30, 1 << 30, 1) if tracked else _lib.View(None, 0, 0, 0)
    args = _lib.StepPagedArgs(64, 16, 1024, 256, _lib.BF16, max_len // 16, max_len, 0, 1e-6, 1e-6, 4096, 1024, None, 4096,
                              *[4096] * 16, _pool(lib, heads=16), 4096, 1, 4096, 4096, 4096, 4096, 4096, weights, 4096, 4096,
                              4096)
    _refused(lib, "sisa_step_paged", args, "too large")


def test_both_steps_refuse_the_same(lib):
    """What sisa_step and sisa_step_paged share is checked once; 64 H that passes 32 bits is no D."""
    from sisa_amd.kernels import _lib
    weights = {n: 4096 for n, t in _lib.StepPagedArgs._fields_ if t is ctypes.c_void_p and n != "res"}
    pool = {n: _lib.View(4096, 1024, 64, 64) for n in ("k", "v", "b")} | {n: _lib.View(4096, 32, 16, 1) for n in ("g", "f")}
    common = dict(B=1, H=2, D=128, FF=256, dtype=_lib.BF16, eps_attn=1e-6, eps_ffn=1e-6, sx=128)
    for bad, word in ((dict(B=0), "B must be"), (dict(B=65), "B must be"), (dict(H=(1 << 26) + 2), "D = 64 H"),
                      (dict(D=64), "D = 64 H"), (dict(H=17, D=1088, sx=1088), "D = 64 H"), (dict(FF=0), "FF positive"),
                      (dict(dtype=_lib.F32), "bf16 or fp16"), (dict(w_gate=None), "given"), (dict(h=4104), "aligned"),
                      (dict(w_down=4100), "w_down"), (dict(sx=120), "x rows"), (dict(res=4104), "x rows"),
                      (dict(b_alpha=None), "null"), (dict(workspace=4112), "256-byte")):
        given = common | weights | bad
        names = {n for n, _ in _lib.StepArgs._fields_}
        step = _lib.StepArgs(**{n: v for n, v in given.items() if n in names}, pos=3, phi_in=4096, phi_out=4096, **pool)
        _refused(lib, "sisa_step", step, word)
        paged = _lib.StepPagedArgs(**given, W=1, max_len=16, pool=_pool(lib))
        _refused(lib, "sisa_step_paged", paged, word)
