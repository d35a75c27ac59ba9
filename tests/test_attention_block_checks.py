"""The launchers around an attention block refuse bad arguments before any device work (no GPU needed)."""
import ctypes as C

import pytest
import torch

from proteinpredictmachinelearning_amd import cabi, ops


@pytest.fixture(scope="module")
def lib():
    return cabi.load()


ONE = C.c_void_p(4096)          # (never read: every call below is refused)


def test_quantizer_and_weight(lib):
    ok = dict(x=ONE, type=0, x_stride=32, q=ONE, q_stride=32, scale=ONE, rows=2, K=32)
    for bad in (dict(x=None), dict(q=None), dict(scale=None), dict(type=3), dict(type=7), dict(rows=0), dict(K=0), dict(K=131072, x_stride=131072, q_stride=131072),
                dict(x_stride=31), dict(q_stride=31)):
        a = dict(ok, **bad)
        assert lib.quantize_rows_i8_hip(a["x"], a["type"], a["x_stride"], a["q"], a["q_stride"], a["scale"], a["rows"], a["K"], None) == 1, bad
    assert b"bad arguments" in lib.ppml_hip_last_error()
    assert [lib.i8_weight_row_bytes_hip(k) for k in (0, 1, 128, 129, 131071, 131072, -5)] == [0, 128, 128, 256, 131072, 0, 0]
    for w, stride, M, K, out in ((None, 32, 2, 32, ONE), (ONE, 32, 2, 32, None), (ONE, 31, 2, 32, ONE), (ONE, 32, 0, 32, ONE), (ONE, 32, 2, 0, ONE)):
        assert lib.i8_weight_pack_hip(w, stride, M, K, out, None) == 1


def test_product(lib):
    need = lib.mul_mat_i8_workspace_hip(5, 30, 600)
    assert need >= 30 * 640 + 120 and [lib.mul_mat_i8_workspace_hip(*s) for s in ((0, 30, 600), (5, 0, 600), (5, 30, 131072), (5, 3, 40))] == [0] * 4
    ok = dict(w=ONE, ws=ONE, x=ONE, xt=0, stride=600, xs=None, bias=None, y=ONE, yt=0, M=5, N=30, K=600, wsp=ONE, nbytes=need)
    for bad in (dict(w=None), dict(ws=None), dict(x=None), dict(y=None), dict(M=0), dict(M=(1 << 22) + 1), dict(N=0), dict(K=0), dict(K=131072, stride=131072), dict(stride=599), dict(yt=3),
                dict(yt=9), dict(xt=5), dict(xt=3), dict(w=C.c_void_p(4097)), dict(wsp=None), dict(nbytes=need - 1), dict(wsp=C.c_void_p(4100))):
        a = dict(ok, **bad)
        assert lib.mul_mat_i8_hip(a["w"], a["ws"], a["x"], a["xt"], a["stride"], a["xs"], a["bias"], a["y"], a["yt"], a["M"], a["N"], a["K"], a["wsp"], a["nbytes"], None) == 1, bad


def desc(**kw):
    a = cabi.QkNormDesc(B=2, L=3, hq=2, hk=1, d=8, rot=8, type=0, eps=1e-6)
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def test_head_norm(lib):
    assert C.sizeof(cabi.QkNormDesc) == 2 * 8 + 8 * 4 + 8 + 18 * 8
    for bad in (dict(B=0), dict(L=0), dict(L=1 << 31), dict(B=1 << 30, L=1 << 30), dict(hq=0, hk=0), dict(hq=-1), dict(hk=65536), dict(d=0), dict(d=513, rot=8), dict(rot=7), dict(rot=10),
                dict(rot=-2), dict(type=3), dict(type=-1), dict(eps=-1.0), dict(eps=float("nan")), dict(position_bytes=2)):
        a = desc(**bad)
        assert lib.qk_norm_rope_hip(C.byref(a), *[ONE] * 8, None) == 1, bad
        assert lib.qk_norm_rope_back_hip(C.byref(a), *[ONE] * 13, 1 << 30, None) == 1, bad
        assert lib.qk_norm_rope_back_workspace_hip(C.byref(a)) == 0
    a = desc(position_bytes=4)
    good = [ONE] * 8                                    # q, k, wq, wk, freqs, positions, q_out, k_out
    for i in (0, 1, 4, 5, 6, 7):
        assert lib.qk_norm_rope_hip(C.byref(a), *[None if j == i else p for j, p in enumerate(good)], None) == 1, i
    assert lib.qk_norm_rope_hip(None, *good, None) == 1
    need = lib.qk_norm_rope_back_workspace_hip(C.byref(a))
    assert need > 0
    good = [ONE] * 13                                   # dq, dk, q, k, wq, wk, freqs, positions, four gradients, workspace
    for i in (0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 12):
        assert lib.qk_norm_rope_back_hip(C.byref(a), *[None if j == i else p for j, p in enumerate(good)], need, None) == 1, i
    assert lib.qk_norm_rope_back_hip(C.byref(a), *good, need - 1, None) == 1


def test_newton_schulz(lib):
    inf = float("inf")
    need = lib.newton_schulz_workspace_hip(2, 30, 40)
    assert need > 0
    assert [lib.newton_schulz_workspace_hip(*s) for s in ((0, 4, 4), (65536, 4, 4), (1, 0, 4), (1, 4, 0), (1, (1 << 20) + 1, 1))] == [0] * 5
    ok = dict(g=ONE, out=ONE, type=0, batch=2, rows=30, cols=40, steps=5, a=1.0, b=1.0, c=1.0, eps=0.0, ws=ONE, nbytes=need)
    for bad in (dict(g=None), dict(out=None), dict(type=3), dict(batch=0), dict(batch=65536), dict(rows=0), dict(cols=0), dict(steps=0), dict(steps=33), dict(a=inf), dict(b=-inf),
                dict(c=float("nan")), dict(eps=-1e-9), dict(eps=inf), dict(a=30.0, b=0.0, c=0.0), dict(steps=32, a=2.0, b=0.0, c=0.0),
                dict(a=8.2, b=-23.6, c=17.3), dict(ws=None), dict(ws=C.c_void_p(4096 + 128)), dict(nbytes=need - 1)):
        a = dict(ok, **bad)
        assert lib.newton_schulz_hip(a["g"], a["out"], a["type"], a["batch"], a["rows"], a["cols"], a["steps"], a["a"], a["b"], a["c"], a["eps"], a["ws"], a["nbytes"], None) == 1, bad


def test_operators_refuse_host_tensors():
    x = torch.zeros(2, 3, 2, 8)
    for call in (lambda: ops.quantize_rows_i8(x), lambda: ops.I8Weight.from_f32(x[0, 0]), lambda: ops.I8Weight(x[0, 0].to(torch.int8), x[0, 0, :, 0]),
                 lambda: ops.qk_norm_rope(x, x), lambda: ops.qk_norm_rope_backward(x, x, x, x), lambda: ops.newton_schulz(x), lambda: ops.mul_mat_i8(x, x)):
        with pytest.raises(TypeError):
            call()
    assert torch.equal(ops.rope_frequencies(4, base=100.0, device="cpu"), torch.tensor([1.0, 0.1], dtype=torch.float64))


def test_the_native_host_side_answers_none_to_what_is_not_ordinary():
    x = torch.zeros(2, 3, 2, 8)
    for name, n in (("mul_mat_i8", 7), ("qk_norm_rope", 8), ("qk_norm_rope_backward", 10), ("newton_schulz", 6)):
        call = getattr(ops._host, name)
        assert call() is None and call(*[None] * n) is None and call(*[x] * n) is None and call(*[1] * n) is None and call(*[None] * 12) is None
    assert ops._host.newton_schulz(x, 5, 1.0, 1.0, 1.0, 1e-7) is None
    assert ops._host.qk_norm_rope(x, x, None, None, None, None, 1e-6, False) is None


def test_counts_past_what_a_launch_can_number(lib):
    """Refused, neither wrapped nor left to the launch: threads along x are counted in 32 bits, tokens of a product in an int."""
    most = 0x7fffffff - 1023
    assert lib.mul_mat_i8_workspace_hip(5, most + 1, 600) == 0 and lib.mul_mat_i8_workspace_hip(5, most, 600) > most * 640
    for n in (most + 1, 0x7fffffff):
        for k in (4, 600):
            assert lib.mul_mat_i8_hip(ONE, ONE, ONE, 0, k, None, None, ONE, 0, 5, n, k, ONE, 1 << 62, None) == 1
            assert b"bad arguments" in lib.ppml_hip_last_error()
    for rows, k in ((1 << 62, 1), (1 << 27, 2048), (1 << 30, 4)):
        assert lib.quantize_rows_i8_hip(ONE, 0, k, ONE, k, ONE, rows, k, None) == 1
        assert b"too many rows" in lib.ppml_hip_last_error()
    for kw in (dict(B=1, L=1 << 27, hq=1, hk=0, d=512, rot=0), dict(B=1 << 16, L=1 << 16, hq=1, hk=1, d=2, rot=2)):
        assert lib.qk_norm_rope_hip(C.byref(desc(**kw)), *[ONE] * 8, None) == 1
        assert b"too many tokens" in lib.ppml_hip_last_error()
