"""Host logic of the token-block operators (rope3d, gated_ffn, quant_rows / gemm_i8) without a GPU: argument checks of
the C ABI (made before any launch, so the made-up addresses are never read), workspace sizes, rotary frequencies, and
the views the wrappers accept as rows or as outputs."""
import math

import pytest
import torch

A = 0x10000          # a made-up, 16-byte aligned device address


def _lib():
    from svk import _lib as L
    return L.load()


def _rope(lib, **kw):
    a = dict(dt=0, q=A, qo=A, heads=2, k=A, ko=A, kv=1, pos=A, pt=0, freqs=A, nt=2, nh=1, nw=1, hd=8, B=1, N=4, il=0)
    a.update(kw)
    return lib.svk_rope3d(a["dt"], a["q"], 16, 64, a["qo"], 16, 64, a["heads"], a["k"], 8, 32, a["ko"], 8, 32, a["kv"],
                          a["pos"], a["pt"], 3, 0, a["freqs"], a["nt"], a["nh"], a["nw"], a["hd"], a["B"], a["N"],
                          a["il"], 0, None)


@pytest.mark.parametrize("kw", [dict(q=None), dict(qo=None), dict(heads=0), dict(k=None), dict(ko=None), dict(kv=-1),
                                dict(pos=None), dict(freqs=None), dict(nt=-1), dict(nt=2 ** 31 - 1, nh=2 ** 31 - 1, nw=4), dict(nt=0, nh=0, nw=0), dict(nt=3),
                                dict(pt=3), dict(B=-1), dict(N=-1), dict(dt=7)])
def test_rope3d_refuses(kw):
    lib = _lib()
    assert _rope(lib, **kw) == -1 and lib.svk_last_error()


def test_rope3d_unsupported_and_empty():
    lib = _lib()
    assert _rope(lib, hd=4098) == -2 and b"head width" in lib.svk_last_error()
    assert _rope(lib, B=65536, N=65536) == -2
    assert _rope(lib, B=0) == 0 and _rope(lib, N=0) == 0          # nothing to launch


def _gated(lib, **kw):
    a = dict(dt=1, x=A, ldx=64, w=A, ldw=64, h=A, ldh=32, M=100, H=32, K=64, act=0, ws=None, n=0)
    a.update(kw)
    return lib.svk_gated_ffn(a["dt"], a["x"], a["ldx"], a["w"], a["ldw"], None, a["h"], a["ldh"], None, a["M"], a["H"],
                             a["K"], a["act"], a["ws"], a["n"], None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(w=None), dict(h=None), dict(ldx=63), dict(ldw=63), dict(ldh=31),
                                dict(M=-1), dict(H=0), dict(K=0), dict(act=3), dict(act=-1), dict(dt=5),
                                dict(K=63, ldx=63, ldw=63)])         # the last: no workspace for the padded rows
def test_gated_ffn_refuses(kw):
    lib = _lib()
    assert _gated(lib, **kw) == -1 and b"svk_gated_ffn" in lib.svk_last_error()


def test_gated_ffn_sizes():
    lib = _lib()
    assert _gated(lib, M=0) == 0
    assert _gated(lib, H=1 << 20, ldh=1 << 20, K=2048, ldx=2048, ldw=2048) == -2      # 8 GiB of weights
    ws = lib.svk_gated_ffn_workspace
    assert ws(1, A, 64, A, 64, 100, 32, 64) == 0
    assert ws(1, A, 63, A, 63, 100, 32, 63) == (100 + 64) * 128      # both padded to 128-byte rows
    assert ws(1, A + 2, 64, A, 64, 100, 32, 64) == 100 * 128         # x misaligned
    from svk import ops
    for M, want in ((8, 0), (ops._FEW, 0), (ops._FEW + 1, (ops._FEW + 65) * 128)):      # few tokens: read as they are
        assert ws(1, A, 63, A, 63, M, 32, 63) == want
        assert (lib.svk_gemm_i8_workspace(A, 63, A, 63, M, 64, 63) == 0) == (want == 0)


@pytest.mark.parametrize("ws,n", [(None, 1 << 30), (A + 8, 1 << 30), (A, (100 + 64) * 128 - 1)])
def test_workspaces_that_are_missing_misaligned_or_short(ws, n):
    lib = _lib()
    odd = dict(K=63, ldx=63, ldw=63)                                 # 100 + 64 rows padded to 128 bytes
    assert _gated(lib, ws=ws, n=n, **odd) == -1 and b"workspace" in lib.svk_last_error()
    assert _i8(lib, K=127, lda=127, ldw=127, N=64, ldy=64, ws=ws, n=n) == -1 and b"workspace" in lib.svk_last_error()


def _gated_bwd(lib, **kw):
    a = dict(dt=0, x=A, w=A, pre=A, dh=A, lddh=32, dx=A, lddx=64, dw=A, db=A, M=100, H=32, K=64, act=0, ws=A, n=1 << 30)
    a.update(kw)
    return lib.svk_gated_ffn_bwd(a["dt"], a["x"], 64, a["w"], 64, a["pre"], a["dh"], a["lddh"], a["dx"], a["lddx"], a["dw"],
                                 a["db"], a["M"], a["H"], a["K"], a["act"], a["ws"], a["n"], None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(w=None), dict(pre=None), dict(dh=None), dict(lddh=31), dict(lddx=63),
                                dict(M=-1), dict(H=0), dict(K=0), dict(act=9), dict(dt=3), dict(ws=None), dict(ws=A + 8),
                                dict(n=100)])
def test_gated_ffn_bwd_refuses(kw):
    lib = _lib()
    assert _gated_bwd(lib, **kw) == -1 and b"svk_gated_ffn_bwd" in lib.svk_last_error()


def test_gated_ffn_bwd_workspace_covers_its_parts():
    lib = _lib()
    for es, dt in ((2, 1), (2, 2), (4, 0)):
        for M, H, K in ((1, 1, 1), (100, 33, 64), (5000, 96, 61), (20000, 40, 72)):
            ld = (2 * H * es + 15) // 16 * 16
            full = lib.svk_gated_ffn_bwd_workspace(dt, A, K, A, K, M, H, K, 1, 1, 1)
            assert full >= M * ld + math.ceil(M / 64) * 2 * H * 4
            assert lib.svk_gated_ffn_bwd_workspace(dt, A, K, A, K, M, H, K, 0, 0, 0) <= full
    assert lib.svk_gated_ffn_bwd_workspace(1, A, 8, A, 8, 0, 8, 8, 1, 1, 1) == 0


def _i8(lib, **kw):
    a = dict(dt=2, a=A, lda=64, sa=A, w=A, ldw=64, sw=A, R=None, ldr=0, y=A, ldy=48, M=100, N=48, K=64, act=0, ws=None, n=0)
    a.update(kw)
    return lib.svk_gemm_i8(a["dt"], a["a"], a["lda"], a["sa"], a["w"], a["ldw"], a["sw"], None, a["R"], a["ldr"], a["y"],
                           a["ldy"], a["M"], a["N"], a["K"], a["act"], a["ws"], a["n"], None)


@pytest.mark.parametrize("kw", [dict(a=None), dict(sa=None), dict(w=None), dict(sw=None), dict(y=None), dict(lda=63),
                                dict(ldw=63), dict(ldy=47), dict(R=A, ldr=47), dict(M=-1), dict(N=0), dict(K=0),
                                dict(K=131072, lda=131072, ldw=131072), dict(act=4), dict(act=-1),
                                dict(lda=65)])                        # the last: rows to be padded, no workspace
def test_gemm_i8_refuses(kw):
    lib = _lib()
    assert _i8(lib, **kw) == -1 and b"svk_gemm_i8" in lib.svk_last_error()


def test_gemm_i8_and_quant_rows_sizes():
    lib = _lib()
    assert _i8(lib, M=0) == 0
    assert _i8(lib, dt=9, M=8) == -1
    assert _i8(lib, N=1 << 20, ldy=1 << 20, K=8192, lda=8192, ldw=8192) == -2
    assert lib.svk_gemm_i8_workspace(A, 61, A, 61, 100, 48, 61) == 148 * 64
    assert lib.svk_gemm_i8_workspace(A, 64, A, 61, 100, 48, 61) == 48 * 64     # aligned tokens may end inside a chunk
    assert lib.svk_gemm_i8_workspace(A, 64, A, 64, 100, 48, 61) == 48 * 64     # the weights' end has to be zeros
    assert lib.svk_gemm_i8_workspace(A + 1, 64, A, 64, 100, 48, 64) == 100 * 64
    assert lib.svk_quant_rows(0, A, 8, A, 8, A, 0, 8, None) == 0
    for bad in ((0, None, 8, A, 8, A, 1, 8), (0, A, 7, A, 8, A, 1, 8), (0, A, 8, A, 7, A, 1, 8), (0, A, 8, A, 8, A, -1, 8),
                (0, A, 8, A, 8, A, 1, 0), (0, A, 8, None, 8, A, 1, 8), (0, A, 8, A, 8, None, 1, 8), (8, A, 8, A, 8, A, 1, 8)):
        assert lib.svk_quant_rows(*bad, None) == -1


def test_rope3d_freqs():
    import svk
    from svk import ops
    f = ops.rope3d_freqs((4, 2, 0), base=100.0, device="cpu")
    assert f.dtype == torch.float64
    assert f.tolist() == pytest.approx([1, 100 ** -0.25, 100 ** -0.5, 100 ** -0.75, 1, 100 ** -0.5], rel=1e-15)
    f = ops.rope3d_freqs((2, 1, 1), base=16.0, shared=True, device="cpu")
    assert f.tolist() == pytest.approx([1, 0.5, 0.25, 0.125], rel=1e-15)
    for bad in ((0, 0, 0), (1, 2), (-1, 2, 2)):
        with pytest.raises(svk.SvkError, match="sections"):
            ops.rope3d_freqs(bad, device="cpu")


def test_no_cpu_path():
    import svk
    from svk import ops
    x = torch.zeros(4, 8)
    for call in (lambda: ops.rope3d(x[None], None, torch.zeros(4, 3), torch.ones(3, dtype=torch.float64), (1, 1, 1), 1),
                 lambda: ops.gated_ffn(x, x), lambda: ops.gated_ffn_bwd(x, x, x, x), lambda: ops.quant_rows(x),
                 lambda: ops.gemm_i8(x.char(), x[:, 0], x.char(), x[:, 0])):
        with pytest.raises(svk.SvkError, match="GPU"):
            call()


def test_token_rows_views():
    import svk
    from svk import ops
    rows = lambda t: ops._token_rows(t, "f", "x")  # noqa: E731
    b = torch.zeros(5, 7, 24)
    assert rows(b) == (35, 24, 24)
    assert rows(b[:, :, 8:16]) == (35, 8, 24)
    assert rows(b[:, -1:]) == (5, 24, 7 * 24)          # the newest token of every batch
    assert rows(b[2, 3]) == (1, 24, 24)
    assert rows(b[:, 3, :8]) == (5, 8, 7 * 24)
    assert rows(b[:1, :1]) == (1, 24, 24)
    assert rows(b[:0])[0] == 0
    for bad in (b[:, :5], b.transpose(0, 1), b.transpose(1, 2), torch.zeros(3, 0), torch.zeros(1, 8).expand(4, 8)):
        with pytest.raises(svk.SvkError):
            rows(bad)


def test_apart_views():
    from svk import ops
    b = torch.zeros(4, 6, 30)
    q, k, v = b[..., :10], b[..., 10:20], b[..., 20:]
    assert ops._apart(q, k) and ops._apart(v, q) and ops._apart(q, q) and ops._apart(q, torch.zeros(4, 6, 10))
    assert ops._apart(b[:2], b[2:]) and ops._apart(q, None) and ops._apart(b[:0], b)
    assert not ops._apart(q, b[..., 5:15]) and not ops._apart(b[..., 5:15], q)
    assert not ops._apart(b[:3], b[1:]) and not ops._apart(b[..., 25:], b.flatten()[5:])
    assert not ops._apart(q, b.view(torch.float16)[..., :10])


def test_rope3d_outputs_in_the_other_input_or_in_the_tables():
    """An output may be its own input only: what it wrote elsewhere would be read as the other input by other threads."""
    import svk
    from svk import ops
    t = torch.zeros(2, 5, 64)
    q, k, new = t[..., :32], t[..., 32:], torch.zeros(2, 5, 32)
    pos = torch.zeros(5, 3)
    assert ops._rope_out(q, k, (q, k), pos)[0] is q                    # in place, packed
    ops._rope_out(q, k, (new, new.clone()), pos)
    ops._rope_out(q, q, (new, new.clone()), pos)                       # the inputs may be one
    ops._rope_out(q, None, (q, None), pos)
    for a in ((q, k, (k, q)), (q, k, (k, new)), (q, k, (new, q)), (q, q, (q, new)), (q, q, (new, q)), (q, k, (new, new)),
              (q, k[..., :16], (k, new[..., :16])), (q, k, (q, k), q[0, :, :3]),
              (q, k, (q, k), pos, t.view(torch.float64).flatten()[-8:])):
        with pytest.raises(svk.SvkError, match="overlaps"):
            ops._rope_out(*a)


B = 0x40000000       # another made-up address


@pytest.mark.parametrize("kw", [dict(qo=B, ko=B), dict(q=B, k=A, qo=A, ko=2 * B), dict(q=A, k=B, qo=2 * B, ko=A),
                                dict(q=A, k=A, qo=A, ko=B), dict(q=A, k=B, qo=B, ko=A),
                                dict(q=A, qo=A, k=B, ko=2 * B, ldqo=32), dict(q=A, qo=2 * B, k=B, ko=B, sbko=64)])
def test_rope3d_entry_refuses_outputs_that_meet(kw):
    lib = _lib()
    a = dict(q=A, qo=2 * B, k=B, ko=3 * B, ldqo=16, sbko=32)
    a.update(kw)
    rc = lib.svk_rope3d(0, a["q"], 16, 64, a["qo"], a["ldqo"], 64, 2, a["k"], 8, 32, a["ko"], 8, a["sbko"], 1, 4 * B, 0, 3, 0, 5 * B,
                        2, 1, 1, 8, 2, 4, 0, 0, None)
    assert rc == -1 and b"overlaps" in lib.svk_last_error()


def test_import_on_a_torch_without_gpu_bindings():
    """A build of torch without GPU support has no raw-stream query; the package imports, and its operators refuse."""
    import os
    import subprocess
    import sys
    import svk
    code = """
import torch
for n in ("_cuda_getCurrentRawStream", "_cuda_getDevice"):
    if hasattr(torch._C, n):
        delattr(torch._C, n)
import svk
try:
    svk.ops.quant_rows(torch.zeros(2, 8))
except svk.SvkError as e:
    print("refused:", e)
"""
    env = dict(os.environ, PYTHONPATH=os.path.dirname(os.path.dirname(os.path.abspath(svk.__file__))))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0 and "no CPU path" in r.stdout, r.stderr


def test_rope3d_outputs_of_either_order_of_batch_and_time():
    import svk
    from svk import ops
    qkv = torch.zeros(5, 2, 96).transpose(0, 1)                        # tokens outside, batches inside
    q, k = qkv[..., :32], qkv[..., 32:64]
    assert ops._rope_out(q, k, (q, k))[1] is k
    ops._rope_out(q, k, (torch.zeros(2, 5, 32), torch.zeros(5, 2, 32).transpose(0, 1)))
    flat = torch.zeros(1000)
    for bad in ((40, 16, 1), (16, 40, 1), (31, 62, 1), (160, 31, 1), (100, 32, 1), (32, 40, 1), (0, 32, 1), (32, 0, 1), (200, 40, 2)):
        with pytest.raises(svk.SvkError, match="rows overlap"):
            ops._rope_out(q, None, (flat.as_strided((2, 5, 32), bad), None))


def test_plan_queries():
    import ctypes
    from svk import ops
    lib = _lib()
    p = (ctypes.c_long * 4)()
    for M in (1, ops._FEW):
        assert lib.svk_gated_ffn_plan(1, 0, M, 32, 64, p) == 0 and list(p) == [0, 1, M, 0]
        assert lib.svk_gemm_i8_plan(M, 32, 64, p) == 0 and list(p) == [0, 1, M, 0]
    for dt in (0, 1, 2):
        for product, rows in ((0, 16384), (1, 16384), (2, 11264)):
            assert lib.svk_gated_ffn_plan(dt, product, 16384, 5632, 2048, p) == 0
            assert p[0] in (64, 128, 256) and p[1] >= 1 and 0 < p[2] <= rows and (p[3] == 0) == (p[2] == rows) and p[3] < p[0]
    assert lib.svk_gemm_i8_plan(16384, 8192, 4096, p) == 0 and list(p) == [256, 1, 16384, 0]
    for bad in ((1, 3, 8, 8, 8), (1, -1, 8, 8, 8), (9, 0, 8, 8, 8), (1, 0, 0, 8, 8), (1, 0, 8, 0, 8), (1, 0, 8, 8, -1)):
        assert lib.svk_gated_ffn_plan(*bad, p) == -1
    assert lib.svk_gated_ffn_plan(1, 0, 8, 8, 8, None) == -1 and lib.svk_gemm_i8_plan(8, 8, 131072, p) == -1


def test_gradient_buffers_to_add_to():
    import svk
    from svk import ops
    x, w = torch.zeros(6, 16), torch.zeros(8, 16)
    dw, db = torch.zeros(8, 16), torch.zeros(8)
    f = lambda g, *others: ops._given(g, (8, 16), -1, "f", "dw", *others)  # noqa: E731
    assert f(True) == (None, True) and f(False) == (None, False) and f(None) == (None, False) and f(1) == (None, True)
    assert f(dw, x, w, None, db)[0] is dw and f(dw, x)[1] is True
    flat = torch.zeros(8 * 16 + 8)
    assert f(flat[:128].view(8, 16), flat[128:])[1] is True
    for bad, others in ((dw.half(), ()), (dw[:7], ()), (dw.flatten(), ()), (torch.zeros(16, 8).t(), ()), (torch.zeros(8, 32)[:, :16], ()),
                        (w, (x, w)), (flat[:128].view(8, 16), (flat[120:128],)), (flat[8:].view(8, 16), (flat[:16],))):
        with pytest.raises(svk.SvkError, match="dw"):
            f(bad, *others)


@pytest.mark.parametrize("add", [4, -1, 8])
def test_gated_ffn_bwd_add_refuses(add):
    lib = _lib()
    rc = lib.svk_gated_ffn_bwd_add(0, A, 64, A, 64, A, A, 32, A, 64, A, A, add, 100, 32, 64, 0, A, 1 << 30, None)
    assert rc == -1 and b"add" in lib.svk_last_error()
