"""CPU tests of the boundary of branched and drafted generation: the header's functions are exported and bound, the argument
structures have the C layout, and entry points and Python calls refuse what they cannot run before anything is launched."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "sisa_hip_branch.h")


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
    assert declared == set(_lib.BRANCH_SIGNATURES) and declared
    assert all(hasattr(lib, name) for name in declared)


def test_struct_layout_matches_c(tmp_path):
    from sisa_amd.kernels import _lib
    pairs = {"PrefixDecodeArgs": "sisa_prefix_decode_args", "VerifyArgs": "sisa_verify_args",
             "StepBranchArgs": "sisa_step_branch_args"}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "sisa_hip_branch.h"', "int main(void) {"]
    expect = []
    for py, c in pairs.items():
        cls = getattr(_lib, py)
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        expect.append(ctypes.sizeof(cls))
        for name, _ in cls._fields_:
            inner = py == "StepBranchArgs" and name in dict(_lib.StepPagedArgs._fields_)
            lines.append(f'printf("%zu\\n", offsetof({c}, {"step." * inner}{name}));')
            expect.append(getattr(cls, name).offset)
    lines += ["return 0;", "}"]
    (tmp_path / "layout.c").write_text("\n".join(lines))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(tmp_path / "layout.c"), "-o", str(exe)],
                   check=True)
    assert [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()] == expect


def _pool(**kw):
    from sisa_amd.kernels import _lib
    row, gate = _lib.View(4096, 2 * 16 * 64, 16 * 64, 64), _lib.View(4096, 32, 16, 1)
    p = dict(pages=2, heads=2, page_size=16, dtype=_lib.BF16, k=row, v=row, b=row, g=gate, f=gate) | kw
    return _lib.PagePoolArgs(*p.values())


def _refused(lib, name, args, word):
    assert getattr(lib, name)(ctypes.byref(args), None) == 1, word
    message = lib.sisa_last_error().decode()
    assert message.startswith(name) and word in message, message


def test_attention_refuses_bad_arguments(lib):
    from sisa_amd.kernels import _lib
    none, row, gate = _lib.View(None, 0, 0, 0), _lib.View(4096, 1024, 64, 64), _lib.View(4096, 32, 16, 1)
    crooked = _lib.View(4104, 1024, 64, 64)
    assert lib.sisa_prefix_decode(None, None) == 1 and lib.sisa_last_error().decode().startswith("sisa_prefix_decode")

    def args(B=2, M=1, W=1, G=1, max_len=16, max_shared=16, out_dtype=0, pool=None, table=4096, lengths=4096, first=4096,
             group=4096, shared=4096, q=row, c=row, gq=gate, fq=gate, lam=4096, out=row, ws=4096):
        return _lib.PrefixDecodeArgs(B, M, W, G, max_len, max_shared, out_dtype, 0, pool or _pool(), table, W, lengths, first,
                                     group, shared, q, c, gq, fq, lam, 1, out, ws)
    for bad, word in ((dict(pool=_pool(page_size=24)), "power of two"), (dict(pool=_pool(g=none)), "no g"), (dict(W=0), "bad shape"),
                      (dict(M=0), "M=0"), (dict(B=-1), "B=-1"), (dict(G=0), "G=0"), (dict(G=3), "G=3"), (dict(max_len=17), "max_len=17"),
                      (dict(max_len=0), "max_len=0"), (dict(max_shared=17), "max_shared=17"), (dict(max_shared=-1), "max_shared=-1"),
                      (dict(out_dtype=_lib.F16), "out_dtype"), (dict(q=crooked), "aligned"), (dict(c=crooked), "aligned"),
                      (dict(gq=none), "gq"), (dict(fq=none), "fq"), (dict(ws=None), "workspace"), (dict(ws=4104), "workspace"),
                      *((dict([(x, None)]), "null pointer") for x in ("table", "lengths", "first", "group", "shared", "lam")),
                      (dict(out=none), "null pointer"),
                      # threads of a launch are counted in 32 bits
                      (dict(B=1 << 27), "too large"), (dict(B=1 << 26, W=1 << 20, max_len=1 << 24, max_shared=0), "too large"),
                      (dict(B=1 << 20, M=128), "too large"), (dict(B=1 << 20, M=1 << 10), "2^28")):
        _refused(lib, "sisa_prefix_decode", args(**bad), word)
    assert lib.sisa_prefix_decode(ctypes.byref(args(B=0)), None) == 0


def test_step_refuses_bad_arguments(lib):
    from sisa_amd.kernels import _lib
    assert lib.sisa_step_branch(None, None) == 1 and lib.sisa_last_error().decode().startswith("sisa_step_branch")
    none = _lib.View(None, 0, 0, 0)

    def args(B=2, M=3, G=1, H=2, D=128, dtype=_lib.BF16, W=1, max_len=16, max_shared=16, row0=0, w_q=4096, pool=None, phi=4096,
             weights=none, first=4096, group=4096, shared=4096, rows=4096, s_rows=4 * 18, ws=4096):
        return _lib.StepBranchArgs(B, H, D, 256, dtype, W, max_len, 0, 1e-6, 1e-6, 4096, D, None, 4096, w_q, *[4096] * 15,
                                   pool or _pool(), 4096, W, 4096, 4096, 4096, 4096, phi, weights, 4096, 4096, ws, M, G, max_shared,
                                   row0, first, group, shared, rows, s_rows)
    for bad, word in ((dict(B=0), "1 .. 64"), (dict(M=0), "1 .. 64"), (dict(B=13, M=5), "1 .. 64"), (dict(B=1 << 30, M=4), "1 .. 64"),
                      (dict(D=192), "B must be"), (dict(dtype=_lib.F32), "bf16 or fp16"), (dict(w_q=None), "given"), (dict(ws=4112), "256-byte"),
                      (dict(pool=_pool(dtype=_lib.F16)), "heads and dtype"), (dict(pool=_pool(heads=3)), "heads and dtype"),
                      (dict(pool=_pool(f=none)), "and f"), (dict(pool=_pool(page_size=20)), "power of two"), (dict(max_len=17), "max_len"),
                      (dict(max_shared=17), "max_shared"), (dict(max_shared=-1), "max_shared"), (dict(G=0), "G=0"), (dict(G=3), "G=3"),
                      (dict(weights=_lib.View(4096, 32, 16, 1)), "tracked"), (dict(row0=-1), "row0"), (dict(s_rows=71), "row0"),
                      (dict(row0=1), "row0"), *((dict([(x, None)]), "null pointer") for x in ("phi", "first", "group", "shared"))):
        _refused(lib, "sisa_step_branch", args(**bad), word)
    size = lib.sisa_step_branch_workspace_bytes
    assert size(0, 2, 128, 256, 1, 1, 16, 0) == size(1, 2, 128, 256, 65, 1, 16, 0) == size(1, 2, 128, 256, 1, 1, 16, -1) == 0
    assert size(2, 2, 128, 256, 4, 1, 600, 500) > size(2, 2, 128, 256, 1, 1, 600, 500) > 0


def test_verification_refuses_bad_arguments(lib):
    from sisa_amd.kernels import _lib
    assert lib.sisa_verify(None, None) == 1 and lib.sisa_last_error().decode().startswith("sisa_verify")

    def args(B=1, K=1, V=8, p_dtype=0, q_dtype=0, p=4096, q=4096, drafts=4096, u=4096, tokens=4096, accepted=4096, ws=4096):
        return _lib.VerifyArgs(B, K, V, p_dtype, q_dtype, 0, p, 16, 8, q, 8, 8, drafts, 1, 1, u, 2, 1, None, tokens, accepted, ws)
    for bad, word in ((dict(B=-1), "bad shape"), (dict(K=-1), "bad shape"), (dict(V=0), "bad shape"), (dict(V=(1 << 24) + 1), "2^24"),
                      (dict(B=(1 << 21) + 1), "2^21"), (dict(p_dtype=_lib.F64), "fp32, bf16 or fp16"), (dict(q_dtype=7), "fp32, bf16 or fp16"),
                      (dict(ws=None), "workspace"), (dict(ws=4104), "workspace"), (dict(B=1 << 20, V=1 << 20), "too large"),
                      *((dict([(x, None)]), "null pointer") for x in ("p", "drafts", "u", "tokens", "accepted"))):
        _refused(lib, "sisa_verify", args(**bad), word)
    assert lib.sisa_verify(ctypes.byref(args(B=0)), None) == 0


def test_workspaces(lib):
    size = lib.sisa_prefix_decode_workspace_bytes
    assert size(0, 1, 1, 1, 1, 0) == size(1, 1, 1, 2, 1, 0) == size(1, 1, 1, 1, 0, 0) == size(1, 1, 1, 1, 1, -1) == 0
    assert size(16, 12, 1, 1, 3000, 2000) > size(16, 12, 1, 1, 3000, 0) > 0


def test_verification_workspace(lib):
    size = lib.sisa_verify_workspace_bytes
    assert size(0, 8) == size(1, 0) == size(1, (1 << 24) + 1) == 0
    assert size(3, 50277) >= 3 * 50 * 16 and size(1, 1) > 0


def test_python_calls_refuse_tensors_off_the_gpu(lib):
    from sisa_amd.kernels import PrefixGroups, sisa_verify_drafts_hip
    with pytest.raises(ValueError, match="GPU"):
        PrefixGroups([1, 2], "cpu")
    with pytest.raises(ValueError, match="at least one group"):
        PrefixGroups([], "cpu")
    p, drafts, u = torch.rand(2, 3, 5), torch.zeros(2, 2, dtype=torch.int64), torch.rand(2, 3)
    with pytest.raises(ValueError, match="GPU"):
        sisa_verify_drafts_hip(p, drafts, u)
    with pytest.raises(ValueError, match="K \\+ 1"):
        sisa_verify_drafts_hip(p[:, :2], drafts, u)


def test_step_refuses_what_its_attention_does(lib):
    """A pool that the attention refuses is refused before the layer's rows are written, not after."""
    from sisa_amd.kernels import _lib
    none, far = _lib.View(None, 0, 0, 0), _lib.View(4096, 1 << 32, 1 << 31, 1 << 26)

    def args(pool):
        return _lib.StepBranchArgs(2, 2, 128, 256, _lib.BF16, 1, 16, 0, 1e-6, 1e-6, 4096, 128, None, 4096, 4096, *[4096] * 15, pool,
                                   4096, 1, 4096, 4096, 4096, 4096, 4096, none, 4096, 4096, 4096, 3, 1, 16, 0, 4096, 4096, 4096, None, 0)
    for bad in (dict(k=far), dict(v=far), dict(b=far), dict(g=_lib.View(4096, 32, 16, 1 << 25)), dict(f=_lib.View(4096, 32, 16, 0)),
                dict(k=_lib.View(4096, 2048, 1024, 56)), dict(b=_lib.View(4096, 2048, 1024, 24))):
        _refused(lib, "sisa_step_branch", args(_pool(**bad)), "a row apart")
