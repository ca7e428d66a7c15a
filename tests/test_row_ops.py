"""CPU: what the row operators refuse, before anything reaches a GPU, and the 64-bit forms that the
GPU tests compare with against known answers."""
import ctypes

import pytest
import torch

import row_reference as ref
from objectdetection_amd import _lib, ops

ARG, WORKSPACE, UNSUPPORTED = -1, -2, -3


def test_reference_8_bit_form_on_known_values():
    v = torch.zeros((2, 130))
    v[0, 0], v[0, 1], v[0, 2] = 448.0, 17.0, 19.0   # 17 lies between 16 and 18, 19 between 18 and 20: to even
    v[0, 128] = 2.0
    v[1, 5] = 450.0
    q, e = ref.quantise(v)
    assert e.tolist() == [[0, -7], [1, 0]]  # 2 = 256 * 2^-7; a block of zeros has e = 0
    assert q[0, :3].tolist() == [448.0, 16.0, 20.0] and q[0, 128] == 256.0
    assert q[1, 5] == 224.0  # 225 lies between 224 and 240
    for dt in ref.MAX8:  # the same values through torch's own conversion
        x = torch.randn((5, 256), generator=torch.Generator().manual_seed(1)) * 3
        q, e = ref.quantise(x, dt)
        s = (2.0 ** e.float()).repeat_interleave(128, 1)
        assert torch.equal(q, (x / s).to(dt).double())
        assert float(q.abs().max()) <= ref.MAX8[dt]


def test_cpu_tensors_are_refused():
    x, w = torch.zeros((4, 8)), torch.zeros((8,))
    w8 = (torch.zeros((3, 8)).to(torch.float8_e4m3fn), torch.zeros((3, 1), dtype=torch.uint8))
    for call in (lambda: ops.rms_norm(x, w), lambda: ops.rms_norm_f8(x, w), lambda: ops.f8_rows(x),
                 lambda: ops.f8_weight_image(x), lambda: ops.f8_linear(x, torch.zeros((3, 8))),
                 lambda: ops.f8_matmul(w8, w8), lambda: ops.grad_norm([x]), lambda: ops.clip_norm_([x], 1.0)):
        with pytest.raises(RuntimeError):
            call()
    assert ops.grad_norm([]).item() == 0.0 and ops.clip_norm_([], 1.0).item() == 0.0
    with pytest.raises(ValueError):
        ops.grad_norm([x], 3.0)
    with pytest.raises(ValueError):
        ops.clip_norm_([x], -1.0)


def _grads(*entries):
    class G(ctypes.Structure):
        _fields_ = [("g", ctypes.c_void_p), ("out", ctypes.c_void_p), ("n", ctypes.c_longlong),
                    ("dtype", ctypes.c_int), ("out_dtype", ctypes.c_int)]
    return (G * len(entries))(*[G(*e) for e in entries])


def test_abi_refuses_bad_gradient_tables():
    L = _lib.lib()
    norm, ws = 4096, 8192  # never touched: every call below is refused on the host
    room = L.lcf_grad_norm_workspace_bytes(2)

    def clip(*entries, p=2, m=1.0, bytes=room, count=None):
        t = _grads(*entries)
        return L.lcf_grad_clip(ctypes.addressof(t), len(entries) if count is None else count, p, m, norm, ws, bytes,
                               None)
    good = (1 << 20, 1 << 21, 100, 0, 0)
    assert clip(good, p=3) == ARG and clip(good, m=-1.0) == ARG and clip(good, m=float("nan")) == ARG
    assert clip(good, count=-1) == ARG
    assert clip((0, 1 << 21, 100, 0, 0)) == ARG and clip((1 << 20, 0, 100, 0, 0)) == ARG
    assert clip((1 << 20, 1 << 21, -1, 0, 0)) == ARG and clip((1 << 20, 1 << 21, 100, 3, 0)) == ARG
    assert clip((1 << 20, 1 << 21, 100, 0, 7)) == ARG
    assert clip(good, bytes=16) == WORKSPACE
    # outputs that overlap another output, a gradient, or their own gradient but not exactly
    assert clip(good, (1 << 22, (1 << 21) + 396, 100, 0, 0)) == ARG
    assert clip(good, ((1 << 21) + 396, 1 << 23, 100, 0, 0)) == ARG
    assert clip((1 << 20, (1 << 20) + 4, 100, 0, 0)) == ARG
    assert clip((1 << 20, 1 << 20, 100, 0, 1)) == ARG
    assert clip((1 << 20, 1 << 20, 100, 0, 0), (1 << 20, 1 << 20, 100, 0, 0)) == ARG
    t = _grads(good)
    assert L.lcf_grad_norm(ctypes.addressof(t), 1, 2, None, ws, room, None) == ARG
    assert L.lcf_grad_norm(ctypes.addressof(t), 1, 2, norm, ws, 8, None) == WORKSPACE


def test_abi_refuses_bad_norm_arguments():
    L = _lib.lib()

    def fwd(x=4096, ldx=64, r=None, ldr=0, rows=4, width=64, dt=0, w=None, wd=0, eps=1e-6, h=None, q8=None, ldq=64,
            s=None, lds=4, fmt=0):
        return L.lcf_rms_norm_fwd(x, ldx, r, ldr, rows, width, dt, w, wd, eps, 8192, h, None, q8, ldq, s, lds, fmt,
                                  None)
    for bad in (dict(x=None), dict(ldx=63), dict(rows=-1), dict(width=0), dict(dt=3), dict(w=4096, wd=9),
                dict(r=4096, ldr=10), dict(h=4096), dict(eps=-1.0), dict(eps=float("nan")), dict(q8=4096),
                dict(q8=4096, s=4096, ldq=40), dict(q8=4100, s=4096), dict(q8=4096, s=4096, lds=3),
                dict(q8=4096, s=4097), dict(q8=4096, s=4096, fmt=2), dict(q8=4096, s=4096, lds=0)):
        assert fwd(**bad) == ARG, bad
    assert fwd(width=16385, ldx=16385) == UNSUPPORTED
    assert fwd(rows=0, x=None) == 0

    def bwd(h=4096, ldh=64, dy=4096, lddy=64, dh=None, lddh=0, rows=4, width=64, dt=0, w=None, wd=0, inv=4096, dx=8192,
            dw=None, ws=None, n=0):
        return L.lcf_rms_norm_bwd(h, ldh, dy, lddy, dh, lddh, rows, width, dt, w, wd, inv, dx, dw, ws, n, None)
    for bad in (dict(h=None), dict(dy=None), dict(inv=None), dict(dx=None), dict(ldh=8), dict(lddy=8),
                dict(dh=4096, lddh=3), dict(rows=-1), dict(width=0), dict(dt=5), dict(dw=4096, wd=4),
                dict(dw=4096)):
        assert bwd(**bad) == ARG, bad
    assert bwd(dw=4096, ws=4096, n=64) == WORKSPACE
    assert bwd(width=20000, ldh=20000, lddy=20000) == UNSUPPORTED


def test_abi_refuses_bad_8_bit_operands():
    L = _lib.lib()

    def quant(x=4096, ldx=64, R=4, C=64, dt=0, fmt=0, sq=0, q=4096, ldq=64, s=4096, lds=4, qt=None, ldqt=0, st=None,
              ldst=0):
        return L.lcf_f8_quant(x, ldx, R, C, dt, fmt, sq, q, ldq, s, lds, qt, ldqt, st, ldst, None, None)
    for bad in (dict(x=None), dict(ldx=10), dict(R=-1), dict(C=-1), dict(dt=7), dict(fmt=2), dict(q=None),
                dict(q=4104), dict(ldq=56), dict(ldq=48), dict(s=None), dict(s=4098), dict(lds=2),
                dict(qt=4096), dict(qt=4096, ldqt=16, st=4096, ldst=3), dict(qt=4096, ldqt=8, st=4096, ldst=4)):
        assert quant(**bad) == ARG, bad
    assert quant(R=0, x=None) == 0 and quant(C=0, x=None) == 0
    assert quant(R=1 << 30, sq=1) == UNSUPPORTED
    last = (1 << 31) - 1  # the end of its last block is past 32 bits
    assert quant(C=last, ldx=last, ldq=1 << 31, lds=1 << 24) == UNSUPPORTED
    assert L.lcf_sum_parts(4096, 1, last, 8192, 0, None) == UNSUPPORTED

    def gemm(a=4096, lda=64, sa=4096, ldsa=4, af=0, b=4096, ldb=64, sb=4096, ldsb=4, bf=0, sq=0, M=4, N=4, K=64,
             out=8192, ldo=4, od=0, ws=None, n=0):
        return L.lcf_f8_gemm(a, lda, sa, ldsa, af, b, ldb, sb, ldsb, bf, sq, M, N, K, None, None, 0, out, ldo, od, ws,
                             n, None)
    for bad in (dict(a=None), dict(lda=60), dict(lda=48), dict(a=4097), dict(sa=None), dict(ldsa=1), dict(af=2),
                dict(b=None), dict(ldb=63), dict(sb=4097), dict(bf=5), dict(M=-1), dict(K=-1), dict(out=None),
                dict(ldo=3), dict(od=3), dict(M=100, K=70000, lda=70016, ldb=70016, ldsa=548, ldsb=548)):
        assert gemm(**bad) == ARG, bad
    assert gemm(M=100, K=70000, lda=70016, ldb=70016, ldsa=548, ldsb=548, ws=4096, n=16) == WORKSPACE
    assert gemm(lda=1 << 23) == UNSUPPORTED and gemm(ldb=1 << 23) == UNSUPPORTED
    for big in (dict(M=last), dict(N=last, ldo=last), dict(M=100, N=last, ldo=last), dict(N=(1 << 25) + 1, ldo=1 << 26),
                dict(M=1 << 30, N=5, ldo=5), dict(M=1 << 20, N=1 << 20, ldo=1 << 20)):
        assert gemm(**big) == UNSUPPORTED, big
    assert L.lcf_f8_gemm_workspace_bytes(last, last, 64, 0) == 0
    assert gemm(M=0, a=None) == 0 and gemm(N=0, b=None) == 0


def test_abi_refuses_bad_weight_gradients():
    L = _lib.lib()

    def grad(x=4096, ldx=64, dy=8192, lddy=32, R=100, K=64, N=32, dt=0, turned=0, dw=12288, dwt=0, db=None, dbt=0,
             ws=16384, n=1 << 30):
        return L.lcf_f8_weight_grad(x, ldx, dy, lddy, R, K, N, dt, turned, dw, dwt, db, dbt, ws, n, None)
    for bad in (dict(x=None), dict(dy=None), dict(dw=None), dict(ldx=60), dict(lddy=31), dict(R=-1), dict(K=-8),
                dict(dt=3), dict(dwt=-1), dict(db=4096, dbt=3), dict(ws=None)):
        assert grad(**bad) == ARG, bad
    for other in (dict(R=0), dict(K=60), dict(N=33, lddy=33), dict(K=264, ldx=264), dict(N=512, lddy=512), dict(x=4098),
                  dict(dt=1, ldx=65), dict(lddy=(1 << 20) + 4)):
        assert grad(**other) == UNSUPPORTED, other
    assert grad(n=100) == WORKSPACE
    assert L.lcf_f8_weight_grad_workspace_bytes(100, 60, 32) == 0
    assert L.lcf_f8_weight_grad_workspace_bytes(100, 64, 32) >= (64 * 32 + 32) * 4


def test_forward_mode_tangents_are_refused():
    """A dual tensor need not require a gradient, and nothing below autograd would carry its tangent."""
    from torch.autograd import forward_ad
    x, w = torch.ones((4, 8)), torch.ones((8,))
    m, b = torch.ones((3, 8)), torch.ones((3,))
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: ops.rms_norm(dual(x), w), lambda: ops.rms_norm(x, dual(w)),
                     lambda: ops.rms_norm(x, w, residual=dual(x)), lambda: ops.f8_linear(dual(x), m),
                     lambda: ops.f8_linear(x, dual(m)), lambda: ops.f8_linear(x, m, dual(b))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_a_change_of_the_build_flags_rebuilds_every_object():
    """Objects are ignored by git and outlive a change of the Makefile's flags: one that keeps the packed
    fp32 instructions would go unnoticed."""
    import os
    import re
    import subprocess
    csrc = os.path.join(os.path.dirname(_lib.__file__), "csrc")
    plan = subprocess.run(["make", "-n", "-W", "Makefile", "-C", csrc], capture_output=True, text=True, check=True).stdout
    sources = re.search(r"^SRCS := ((?:.*\\\n)*.*)$", open(os.path.join(csrc, "Makefile")).read(), re.M).group(1)
    sources = sources.replace("\\", " ").split()
    assert len(sources) >= 12
    for source in sources:
        line = next(k for k in plan.splitlines() if f"-c {source} " in k)
        assert "-packed-fp32-ops" in line
    assert "-o ../_row_ops.so" in plan and "-o ../liblcf_cpu.so" in plan and "-o ../liblcf.so" in plan


def test_long_sums_of_few_rows_are_split_where_there_is_room():
    """A weight gradient of few channels is few rows over a long sum: without a split 13 workgroups walk
    all of it.  The room is offered, not asked for."""
    L = _lib.lib()
    for M, N, K in ((50, 200, 136000), (64, 512, 136000), (18, 128, 136000), (64, 260, 136000), (8, 16, 90000),
                    (40, 64, 70000), (17, 1000, 8192), (33, 24, 4096), (16, 8192, 8193)):
        for t in range(3):
            assert L.lcf_f8_gemm_workspace_bytes(M, N, K, t) == 0
            parts, rest = divmod(L.lcf_f8_gemm_split_bytes(M, N, K, t), M * N * 4)
            assert rest == 0 and 2 <= parts <= 256, (M, N, K, t, parts)
    for M, N, K in ((8, 8192, 4096), (1, 4096, 8192), (64, 256, 2048), (32, 64, 4096), (16, 8200, 30000)):
        assert L.lcf_f8_gemm_split_bytes(M, N, K, 0) == 0
    for M, N, K in ((65, 200, 136000), (100, 64, 9000), (8192, 4096, 8192)):  # many rows need what they are offered
        assert L.lcf_f8_gemm_split_bytes(M, N, K, 0) == L.lcf_f8_gemm_workspace_bytes(M, N, K, 0)
    last = (1 << 31) - 1
    assert L.lcf_f8_gemm_split_bytes(last, last, 64, 0) == 0 and L.lcf_f8_gemm_split_bytes(0, 5, 64, 0) == 0


def test_rms_norm_module_takes_what_nn_rms_norm_takes():
    from torch import nn

    from objectdetection_amd import spconv
    for kw in (dict(), dict(eps=1e-5), dict(elementwise_affine=False), dict(device="cpu", dtype=torch.bfloat16)):
        a, b = spconv.RMSNorm(24, **kw), nn.RMSNorm(24, **kw)
        assert a.eps == b.eps and list(a.state_dict()) == list(b.state_dict())
        assert a.weight is b.weight is None or (a.weight.dtype == b.weight.dtype and torch.equal(a.weight, b.weight))
