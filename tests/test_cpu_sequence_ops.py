"""Refusals of the sequence-network operators and of their C entry points: every one comes from the
host, before anything is launched."""
import ctypes as C

import pytest
import torch

import kalman_vae_amd as kv
from kalman_vae_amd import _capi as capi


E8 = lambda *s: torch.zeros(s, dtype=torch.float8_e4m3fn)  # noqa: E731
ONE = lambda *s: torch.ones(s)  # noqa: E731


def test_no_cpu_path():
    u, w = torch.zeros(3, 2, 12), torch.ones(12)
    for call in (lambda: kv.gated_scan(u), lambda: kv.gated_scan_step(u[0], torch.zeros(2, 4)),
                 lambda: kv.rms_norm(u, w), lambda: kv.rms_norm_quantized(u, w), lambda: kv.quantize_rows(u)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def as_if_on_gpu(monkeypatch):
    """The argument checks run on any tensor; what follows them is not reached in these tests."""
    from kalman_vae_amd import sequence_ops
    monkeypatch.setattr(sequence_ops, "_device_of", lambda *t: torch.device("cpu"))


@pytest.mark.parametrize("call,error,match", [
    (lambda: kv.gated_scan(torch.zeros(3, 12)), ValueError, "shape"),
    (lambda: kv.gated_scan(torch.zeros(3, 2, 13)), ValueError, "3 equal parts"),
    (lambda: kv.gated_scan(torch.zeros(3, 2, 13), output_gate=False), ValueError, "2 equal parts"),
    (lambda: kv.gated_scan(torch.zeros(3, 2, 12).double()), TypeError, "float64"),
    (lambda: kv.gated_scan(torch.zeros(3, 2, 12), torch.zeros(2, 5)), ValueError, "h0 must have shape"),
    (lambda: kv.gated_scan(torch.zeros(3, 2, 12), torch.zeros(2, 4).half()), TypeError, "float32"),
    (lambda: kv.gated_scan(torch.zeros(3, 2, 12), mask=torch.zeros(2, 3)), ValueError, "mask must have"),
    (lambda: kv.gated_scan_step(torch.zeros(3, 2, 12), torch.zeros(2, 4)), ValueError, "shape"),
    (lambda: kv.gated_scan_step(torch.zeros(2, 12), torch.zeros(2, 8)[:, ::2]), ValueError, "contiguous"),
    (lambda: kv.gated_scan_step(torch.zeros(2, 12), torch.zeros(2, 4), mask=torch.zeros(3)), ValueError, "mask"),
    (lambda: kv.gated_scan_step(torch.zeros(2, 12, requires_grad=True), torch.zeros(2, 4)), RuntimeError, "no gradient"),
    (lambda: kv.rms_norm(torch.zeros(3, 4), torch.ones(5)), ValueError, "weight must have shape"),
    (lambda: kv.rms_norm(torch.zeros(3, 4), torch.ones(4).half()), TypeError, "weight must be"),
    (lambda: kv.rms_norm(torch.zeros(()), torch.ones(4)), ValueError, "one axis"),
    (lambda: kv.rms_norm(torch.zeros(3, 4).long(), torch.ones(4)), TypeError, "int64"),
    (lambda: kv.rms_norm(torch.zeros(3, 4), torch.ones(4), residual=torch.zeros(4)), ValueError, "residual"),
    (lambda: kv.rms_norm(torch.zeros(3, 4), torch.ones(4), residual=torch.zeros(3, 4).half()), TypeError, "residual"),
    (lambda: kv.rms_norm(torch.zeros(1, 16385), torch.ones(16385)), NotImplementedError, "16384"),
    (lambda: kv.rms_norm_quantized(torch.zeros(3, 4), torch.ones(4, requires_grad=True)), RuntimeError, "no gradient"),
    (lambda: kv.quantize_rows(torch.zeros(3, 4, requires_grad=True)), RuntimeError, "no gradient"),
    (lambda: kv.quantize_rows(torch.zeros(1, 16385)), NotImplementedError, "16384"),
    (lambda: kv.linear_8bit(torch.zeros(2, 4), ONE(2), E8(3, 4), ONE(3)), TypeError, "x must be"),
    (lambda: kv.linear_8bit(E8(2, 4), ONE(2), torch.zeros(3, 4), ONE(3)), TypeError, "weight must be"),
    (lambda: kv.linear_8bit(E8(2, 4), ONE(2).half(), E8(3, 4), ONE(3)), TypeError, "x_scale must be"),
    (lambda: kv.linear_8bit(E8(2, 4), ONE(2), E8(3, 5), ONE(3)), ValueError, "expected"),
    (lambda: kv.linear_8bit(E8(2, 4), ONE(3), E8(3, 4), ONE(3)), ValueError, "one scale per row"),
    (lambda: kv.linear_8bit(E8(2, 4), ONE(2), E8(3, 4), ONE(3, 1)), ValueError, "one scale per row"),
    (lambda: kv.linear_8bit(E8(2, 4), ONE(2), E8(3, 4), ONE(3), bias=ONE(4)), ValueError, "bias must have"),
    (lambda: kv.linear_8bit(E8(2, 4), ONE(2), E8(3, 4), ONE(3), dtype=torch.float64), TypeError, "float64"),
    (lambda: kv.linear_8bit(E8(2, 4), ONE(2).requires_grad_(), E8(3, 4), ONE(3)), RuntimeError, "no gradient"),
])
def test_refusals(monkeypatch, call, error, match):
    as_if_on_gpu(monkeypatch)
    with pytest.raises(error, match=match):
        call()


def test_c_entry_points_refuse_before_launching():
    lib = capi.load()
    one = 4096                                   # an address that is never followed
    d = capi.GatedScan(T=4, B=2, H=8, dtype=capi.KVAE_F32, gated=1)
    assert lib.kvae_gated_scan_forward(C.byref(d), None, 0, None) == -1            # no u
    d.u = one
    assert lib.kvae_gated_scan_forward(C.byref(d), None, 0, None) == -1            # no y
    d.y, d.dtype = one, capi.KVAE_F64
    assert lib.kvae_gated_scan_forward(C.byref(d), None, 0, None) == -2
    d.dtype, d.T = capi.KVAE_F32, 0
    assert lib.kvae_gated_scan_forward(C.byref(d), None, 0, None) == -1
    d.T = 1 << 20                                # cut into segments: needs a workspace
    need = lib.kvae_gated_scan_workspace_bytes(d.T, d.B, d.H, d.dtype)
    assert need > 0 and lib.kvae_gated_scan_forward(C.byref(d), one, need - 1, None) == -3
    assert lib.kvae_gated_scan_backward(C.byref(d), one, need, None) == -1         # no states, dy, du
    d.T, d.B, d.H = 1, 1 << 30, 1 << 20
    assert lib.kvae_gated_scan_forward(C.byref(d), None, 0, None) == -5
    assert lib.kvae_gated_scan_forward(None, None, 0, None) == -1
    assert lib.kvae_gated_scan_step(2, 8, 9, 1, one, 24, None, 0, one, one, None) == -2
    assert lib.kvae_gated_scan_step(2, 8, 0, 1, None, 24, None, 0, one, one, None) == -1
    n = capi.RmsNorm(rows=2, D=8, dtype=capi.KVAE_F32, weight_dtype=capi.KVAE_F32, x=one, weight=one)
    assert lib.kvae_rms_norm_forward(C.byref(n), None) == -1                       # no y
    n.y = one
    assert lib.kvae_rms_norm_quantized(C.byref(n), None) == -1                     # no scale
    assert lib.kvae_rms_norm_backward(C.byref(n), None) == -1
    n.weight_dtype = capi.KVAE_BF16
    assert lib.kvae_rms_norm_forward(C.byref(n), None) == -2
    n.weight_dtype, n.D = capi.KVAE_F32, 16385
    assert lib.kvae_rms_norm_forward(C.byref(n), None) == -2
    n.D, n.rows = 8, 1 << 32
    assert lib.kvae_rms_norm_forward(C.byref(n), None) == -5
    assert lib.kvae_quantize_rows(2, 8, 1, one, 8, one, one, None) == -2
    assert lib.kvae_quantize_rows(2, 8, 0, one, 8, None, one, None) == -1
    assert lib.kvae_linear_8bit(2, 8, 0, one, one, one, one, None, 0, one, None) == -1
    assert lib.kvae_linear_8bit(2, 8, 4, one, None, one, one, None, 0, one, None) == -1
    assert lib.kvae_linear_8bit(2, 8, 4, one, one, one, one, None, 1, one, None) == -2
    assert lib.kvae_linear_8bit(2, 1 << 31, 4, one, one, one, one, None, 0, one, None) == -5
    assert lib.kvae_linear_8bit(2, 4, (1 << 22) + 1, one, one, one, one, None, 0, one, None) == -5
    assert lib.kvae_linear_8bit((1 << 31) + 1, 4, 4, one, one, one, one, None, 0, one, None) == -5


def test_segments_of_the_time_axis():
    """The workspace says how the time axis is cut: not at all for short sequences or many channels,
    into at most 128 segments, none of fewer than two rounds of a workgroup (4 chunks of 8 or 16 steps)."""
    lib = capi.load()
    size = lambda T, B, H, d=0: lib.kvae_gated_scan_workspace_bytes(T, B, H, d)  # noqa: E731
    assert size(1, 1, 1) == size(255, 1, 1) == size(127, 1, 1, 2) == size(1000, 4096, 128) == 0
    for T in (256, 600, 1000, 32768, 1 << 22):
        for B, H, d in ((1, 1, 0), (1, 520, 3), (3, 65, 2)):
            segs = size(T, B, H, d) / (8 * B * H)
            assert segs == int(segs) and segs <= min(128, T / (64 if d else 128)), (T, B, H, d)
    assert size(1 << 22, 1, 1) == 128 * 8


def test_ctypes_structs_match_header(tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = {"kvae_gated_scan": (capi.GatedScan, "dh0"), "kvae_rms_norm": (capi.RmsNorm, "dweight"),
             "kvae_adamw": (capi.AdamW, "lr_device")}
    src = '#include <stdio.h>\n#include "kvae_kalman.h"\nint main(void){\n'
    for n, (_, last) in names.items():
        src += f'printf("%zu %zu\\n", sizeof({n}), offsetof({n}, {last}));\n'
    (tmp_path / "s.c").write_text(src + "return 0;}\n")
    subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")])
    lines = subprocess.check_output([str(tmp_path / "s")], text=True).splitlines()
    for line, (cls, last) in zip(lines, names.values()):
        assert line == f"{C.sizeof(cls)} {getattr(cls, last).offset}"


def test_adamw_refusals():
    from kalman_vae_amd import AdamW, adamw_step
    z = lambda n=4, d=torch.float32: torch.zeros(n, dtype=d)  # noqa: E731
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        adamw_step([z()], [z()], [z()], [z()], 1)
    p = z()
    codes, scale = z(4, torch.float8_e4m3fn), z(1)
    for args, error, match in [
            (([p], [z(5)], [z()], [z()], 1), ValueError, "elements"),
            (([p], [z().double()], [z()], [z()], 1), TypeError, "Double"),
            (([z().double()], [z()], [z()], [z()], 1), TypeError, "Double"),
            (([p], [], [z()], [z()], 1), ValueError, "0 gradients for 1"),
            (([p], [z()], [z().half()], [z()], 1), TypeError, "exp_avgs"),
            (([p], [z(8)[::2]], [z()], [z()], 1), ValueError, "contiguous"),
            (([p, p], [z(), z()], [z(), z()], [z(), z()], 1), ValueError, "twice"),
            (([p], [z()], [z()], [z()], 0), ValueError, "counts from 1"),
            (([p], [z()], [z()], [z()], torch.zeros(1)), ValueError, "int64"),
            (([p], [z()], [(codes, scale)], [z()], 1), TypeError, "all float32"),
            (([p], [z()], [(codes, z(2))], [(codes, scale)], 1), ValueError, "1 scales"),
            (([p], [z()], [(z(), scale)], [(codes, scale)], 1), TypeError, "Float8"),
            ((p, [z()], [z()], [z()], 1), TypeError, "list"),
            (([p], [z()], [(codes,)], [(codes, scale)], 1), TypeError, "pairs"),
    ]:
        with pytest.raises(error, match=match):
            adamw_step(*args)
    with pytest.raises(ValueError, match="masters"):
        adamw_step([p], [z()], [z()], [z()], 1, masters=[z()])
    with pytest.raises(ValueError, match="lr as a tensor"):
        adamw_step([p], [z()], [z()], [z()], 1, lr=torch.ones(1))
    q = torch.nn.Parameter(p)
    for kw in (dict(lr=-1), dict(betas=(1.0, 0.9)), dict(eps=-1), dict(weight_decay=-1), dict(state_bits=4),
               dict(lr=torch.ones(1))):
        with pytest.raises(ValueError):
            AdamW([q], **kw)


def test_adamw_c_entry_point_refuses_before_launching():
    lib, one = capi.load(), 4096
    row = lambda numel=4, master=0, scale=0: [numel, one, one, one, one, scale, scale, master]  # noqa: E731

    def call(rows, **kw):
        table = (C.c_int64 * (8 * max(1, len(rows))))(*[v for r in rows for v in r])
        d = capi.AdamW(**{**dict(count=len(rows), state_bits=32, step=1, beta1=0.9, beta2=0.999), **kw})
        d.tensors = C.addressof(table)
        return lib.kvae_adamw_step(C.byref(d), None)

    assert call([]) == -1 and call([row()] * 49) == -1 and call([row(0)]) == -1
    assert call([row()], step=0) == -1 and call([row(), row(master=one)]) == -1
    assert call([row()], state_bits=8) == -1                     # no scales
    assert call([row()], state_bits=4) == -2 and call([row()], dtype=capi.KVAE_F64) == -2
    assert lib.kvae_adamw_step(None, None) == -1
    assert call([row(1 << 45)]) == -5


def test_limits_of_a_launch_are_refused():
    """A launch has fewer than 2^32 threads and its lanes 32-bit offsets: what does not fit is refused
    before anything is launched, whatever the addresses (never followed here)."""
    lib, one = capi.load(), 4096
    d = capi.GatedScan(T=1, B=1 << 31, H=2, dtype=capi.KVAE_F32, gated=1, u=one, y=one, u_stride_b=6, u_stride_t=6)
    assert lib.kvae_gated_scan_forward(C.byref(d), None, 0, None) == -5
    assert lib.kvae_gated_scan_step(1 << 31, 2, 0, 1, one, 6, None, 0, one, one, None) == -5
    for code, size in ((capi.KVAE_F32, 4), (capi.KVAE_BF16, 2)):
        for name, width in (("u", size), ("mask", 1)):
            d = capi.GatedScan(T=1, B=2, H=2, dtype=code, gated=1, u=one, y=one, mask=one, u_stride_b=6, u_stride_t=6)
            setattr(d, name + "_stride_b", (1 << 31) // width + 1)
            assert lib.kvae_gated_scan_forward(C.byref(d), None, 0, None) == -5, name
    d = capi.GatedScan(T=1 << 20, B=2, H=8, dtype=capi.KVAE_F32, gated=1, u=one, y=one, u_stride_b=24, u_stride_t=48)
    need = lib.kvae_gated_scan_workspace_bytes(d.T, d.B, d.H, d.dtype)
    assert lib.kvae_gated_scan_forward(C.byref(d), None, need, None) == -3
    assert lib.kvae_linear_8bit(2, (1 << 26) + 1, 4, one, one, one, one, None, 0, one, None) == -5
    assert lib.kvae_linear_8bit(1 << 20, 1 << 21, 4, one, one, one, one, None, 0, one, None) == -5
    assert lib.kvae_quantize_rows(1 << 31, 8, 0, one, 8, one, one, None) == -5


def test_adamw_refuses_memory_that_is_written_twice():
    from kalman_vae_amd import adamw_step
    z = lambda n=4: torch.zeros(n)  # noqa: E731
    flat, state = z(10), z()
    for args in (([flat[:4], flat[3:7]], [z(), z()], [z(), z()], [z(), z()], 1),       # views that overlap
                 ([z(), z()], [z(), z()], [state, state], [z(), z()], 1),              # one state for two
                 ([z()], [z()], [state], [state], 1),                                  # m and v the same
                 ([state], [z()], [state], [z()], 1)):                                 # m is the parameter
        with pytest.raises(ValueError, match="share memory"):
            adamw_step(*args)
    with pytest.raises(RuntimeError, match="no CPU fallback"):                         # neighbours are fine
        adamw_step([flat[:4], flat[4:8]], [z(), z()], [z(), z()], [z(), z()], 1)
