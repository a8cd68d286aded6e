"""What the operators of a block that answers token by token refuse, without a GPU: the C entry points before any device call, the
tensor functions by type, shape and place."""
import shutil
import subprocess
import sys

import pytest
import torch

BF = torch.bfloat16


@pytest.fixture
def lib():
    from katz_amd import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("libkatz_hip.so not built")
    return _lib.load()


def test_block_norm_entry_point(lib):
    def call(y=16, h=16, gate=None, gate_rows=1, post=(None, None), pre=(None, None), ho=16, u=16, M=4, D=64, flags=0, t=0, st=0):
        return lib.kh_block_norm(y, h, gate, gate_rows, *post, *pre, ho, u, M, D, 1.0, 1e-6, flags, t, st, None)

    assert call(h=None) == -1 and call(M=0) == -1 and call(D=0) == -1
    assert call(ho=None) == -1                              # y without a place for the sum
    assert call(y=None) == -1 and call(y=None, ho=None, u=None) == -1
    assert call(y=None, ho=None, flags=2) == -1             # nothing to norm
    assert call(y=None, ho=None, gate=16) == -1
    assert call(post=(16, None)) == -1                      # weights of a norm that is not asked for
    assert call(u=None, pre=(16, None)) == -1
    assert call(gate=16, gate_rows=0) == -1 and call(gate=16, gate_rows=3) == -1 and call(gate=16, gate_rows=5) == -1
    assert call(flags=4) == -1 and call(t=3) == -1 and call(st=-1) == -1
    assert call(t=0, st=1) == -2 and call(t=2, st=0) == -2  # the stream has y's type or 32 bits
    assert call(D=32769) == -4 and call(M=1 << 31) == -4


def test_w4_entry_points(lib):
    quant = lambda w=16, q=16, s=16, N=4, K=64, g=64, t=0: lib.kh_quantize_w4(w, q, s, None, N, K, g, t, None)      # noqa: E731
    assert quant(w=None) == -1 and quant(N=0) == -1 and quant(K=0) == -1 and quant(t=3) == -1
    assert quant(g=16) == -2 and quant(g=96) == -2 and quant(q=8) == -3 and quant(s=2) == -3 and quant(K=(1 << 24) + 1) == -4
    value = lambda q=16, o=16, N=4, K=64, g=64, t=0: lib.kh_dequantize_w4(q, 16, None, o, N, K, g, t, None)         # noqa: E731
    assert value(q=None) == -1 and value(o=None) == -1 and value(N=0) == -1 and value(t=-1) == -1 and value(g=0) == -2 and value(q=24) == -3

    def linear(x=16, q=16, s=16, a=None, b=None, c=None, ws=None, y=16, M=2, N=8, K=64, R=0, g=64, t=0):
        return lib.kh_w4_linear(x, q, s, None, None, a, b, c, None, y, ws, M, N, K, R, g, t, None)

    assert linear(x=None) == -1 and linear(y=None) == -1 and linear(M=0) == -1 and linear(N=-1) == -1 and linear(t=2) == -1
    assert linear(R=32) == -1 and linear(R=32, a=16, b=16, c=16, K=8192) == -1          # operands, workspace missing
    assert linear(R=40, a=16, b=16, c=16, ws=16) == -2 and linear(R=160, a=16, b=16, c=16, ws=16) == -4
    assert linear(g=48) == -2 and linear(q=4) == -3 and linear(M=1 << 21) == -4
    size = lib.kh_w4_linear_workspace_bytes
    assert size(4, 1280, 0) == 0 and size(4, 1280, 64) == 0 and size(4, 8192, 64) >= 4 * 64 * 4 and size(40, 1280, 64) >= 40 * 64 * 4 and size(4, 1280, 48) == -1 and size(0, 1280, 32) == -1 and size(1, 64, 160) == -1


def test_linear_attention_entry_points(lib):
    def prompt(q=16, g=16, s=16, so=16, slots=None, n=2, seg=None, rows=0, ws=16, B=2, H=4, Hk=2, T=100, dk=64, dv=64, ld=256, bs=25600, o=16):
        return lib.kh_linear_attention_bf16(q, 16, 16, o, g, s, so, slots, n, seg, rows, ws, B, H, Hk, T, dk, dv, *([ld] * 4), *([bs] * 4), 0.1, None)

    assert prompt(q=None) == -1 and prompt(g=None) == -1 and prompt(so=None) == -1 and prompt(B=0) == -1 and prompt(T=0) == -1
    assert prompt(H=4, Hk=3) == -1 and prompt(Hk=0) == -1 and prompt(n=1) == -1 and prompt(n=0, slots=16) == -1 and prompt(ld=248) == -1
    assert prompt(seg=16, rows=-1) == -1 and prompt(T=1000, ws=None) == -1
    assert prompt(dk=32) == -2 and prompt(dv=96) == -2 and prompt(dv=1088, ld=8192) == -2
    assert prompt(ld=260) == -3 and prompt(q=8) == -3 and prompt(so=4) == -3 and prompt(ws=8) == -3
    assert prompt(T=1 << 31) == -4 and prompt(n=1 << 31) == -4
    size = lib.kh_linear_attention_workspace_bytes
    assert size(2, 4, 0, 1, 64, 64) == -1 and size(2, 4, 10, 20, 80, 64) == -2 and size(2, 4, 64, 128, 64, 64) == 0
    assert size(1, 1, 1 << 20, 1 << 20, 128, 128) > 0 and size(1 << 21, 1, 1, 1 << 21, 64, 64) == -4

    def step(s=16, so=16, B=2, dk=64, ld=256, n=2, flags=0):
        return lib.kh_linear_attention_step_bf16(16, 16, 16, 16, 16, s, so, None, n, B, 4, 4, dk, 64, *([ld] * 4), 0.1, flags, None)

    assert step(s=None) == -1 and step(so=None) == -1 and step(B=0) == -1 and step(n=1) == -1 and step(ld=128) == -1
    assert step(flags=2) == -1 and step(dk=96) == -2 and step(ld=258) == -3


def test_tensor_functions_refuse_what_is_not_on_the_gpu(lib):
    from katz_amd import ops
    from katz_amd._lib import KatzHipError

    x = torch.zeros(4, 64, dtype=BF)
    for call in (lambda: ops.block_norm(x, x), lambda: ops.quantize_w4(x), lambda: ops.linear_attention_step(x, x, x, 1, torch.zeros(1), torch.zeros(4, 1, 64, 64)),
                 lambda: ops.linear_attention(x[None], x[None], x[None], 1, torch.zeros(1)),
                 lambda: ops.w4_linear(x, ops.W4Weight(torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 4, dtype=BF), None, 64, 64)),
                 lambda: ops.dequantize_w4(ops.W4Weight(torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 4, dtype=BF), None, 64, 64))):
        with pytest.raises((KatzHipError, RuntimeError)):
            call()


def test_w4_weight_checks_its_parts():
    from katz_amd.ops import W4Weight

    q, s, z = torch.zeros(8, 48, dtype=torch.uint8), torch.zeros(8, 4, dtype=BF), torch.zeros(8, 4, dtype=torch.uint8)
    w = W4Weight(q, s, z, 70, 32)
    assert (w.out_features, w.in_features, w.groups) == (8, 70, 3)
    for bad in (lambda: W4Weight(q, s, z, 70, 16), lambda: W4Weight(q, s, z, 100, 32), lambda: W4Weight(q, s[:, :3], z, 70, 32),
                lambda: W4Weight(q[:4], s, z, 70, 32), lambda: W4Weight(q, s, z[:, :2], 70, 32), lambda: W4Weight(q, s, z, 0, 32),
                lambda: W4Weight(q.t().contiguous().t(), s, z, 70, 32)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: W4Weight(q.to(torch.int8), s, z, 70, 32), lambda: W4Weight(q, s.float(), z, 70, 32), lambda: W4Weight(q, s, s, 70, 32)):
        with pytest.raises(TypeError):
            bad()


@pytest.mark.gpu
def test_tensor_functions_refuse_shapes_and_types():
    from katz_amd import ops
    from katz_amd._lib import KatzHipError

    d = "cuda:0"
    t = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype, device=d)      # noqa: E731
    w = ops.quantize_w4(t(8, 64), 64)
    bad = [
        (ValueError, lambda: ops.block_norm(t(2, 3, 64), t(2, 3, 32))),
        (ValueError, lambda: ops.block_norm(t(2, 3, 64), t(2, 3, 64), gate=t(3, 64))),
        (ValueError, lambda: ops.block_norm(t(2, 3, 64), t(2, 3, 64), kind="group")),
        (ValueError, lambda: ops.block_norm(t(2, 3, 64), t(2, 3, 64), post_weight=t(64))),
        (ValueError, lambda: ops.block_norm(t(2, 3, 64), t(2, 3, 64), pre=False, pre_weight=t(64))),
        (ValueError, lambda: ops.block_norm(None, t(2, 64), gate=t(64))),
        (ValueError, lambda: ops.block_norm(t(2, 64), t(2, 64), pre_weight=t(32))),
        (ValueError, lambda: ops.block_norm(t(64, 2).t(), t(2, 64))),
        (TypeError, lambda: ops.block_norm(t(2, 64, dtype=torch.float32), t(2, 64))),
        (TypeError, lambda: ops.block_norm(t(2, 64), t(2, 64), gate=t(64, dtype=torch.float32))),
        (KatzHipError, lambda: ops.block_norm(t(1, 40000), t(1, 40000))),
        (KatzHipError, lambda: ops.block_norm(t(2, 64), torch.zeros(2, 64, dtype=BF))),
        (ValueError, lambda: ops.quantize_w4(t(8, 64), 48)),
        (TypeError, lambda: ops.quantize_w4(t(8, 64, dtype=torch.float64))),
        (ValueError, lambda: ops.quantize_w4(t(64, 8).t())),
        (TypeError, lambda: ops.dequantize_w4(w, torch.float64)),
        (ValueError, lambda: ops.w4_linear(t(2, 32), w)),
        (TypeError, lambda: ops.w4_linear(t(2, 64, dtype=torch.float32), w)),
        (TypeError, lambda: ops.w4_linear(t(2, 64), w, t(8, dtype=torch.float32))),
        (ValueError, lambda: ops.w4_linear(t(2, 64), w, t(9))),
        (ValueError, lambda: ops.w4_linear(t(2, 64), w, None, t(32, 64))),
        (ValueError, lambda: ops.w4_linear(t(2, 64), w, None, t(40, 64), t(8, 40), t(40, dtype=torch.float32))),
        (ValueError, lambda: ops.w4_linear(t(2, 64), w, None, t(160, 64), t(8, 160), t(160, dtype=torch.float32))),
        (ValueError, lambda: ops.w4_linear(t(2, 64), w, residual=t(2, 9))),
        (ValueError, lambda: ops.w4_linear(t(4, 64)[::2], w)),
    ]
    g, f = t(2, dtype=torch.float32), torch.float32
    bad += [
        (ValueError, lambda: ops.linear_attention(t(1, 4, 128), t(1, 4, 128), t(1, 4, 128), 3, g)),
        (ValueError, lambda: ops.linear_attention(t(1, 4, 128), t(1, 5, 128), t(1, 4, 128), 2, g)),
        (ValueError, lambda: ops.linear_attention(t(1, 4, 128), t(1, 4, 64), t(1, 4, 128), 2, g)),
        (TypeError, lambda: ops.linear_attention(t(1, 4, 128, dtype=f), t(1, 4, 128), t(1, 4, 128), 2, g)),
        (TypeError, lambda: ops.linear_attention(t(4, 128), t(4, 128), t(4, 128), 2, g)),
        (ValueError, lambda: ops.linear_attention(t(1, 4, 128), t(1, 4, 128), t(1, 4, 128), 2, t(3, dtype=f))),
        (ValueError, lambda: ops.linear_attention(t(1, 4, 128), t(1, 4, 128), t(1, 4, 128), 2, g, state=t(2, 2, 64, 64, dtype=f))),
        (ValueError, lambda: ops.linear_attention(t(1, 4, 128), t(1, 4, 128), t(1, 4, 128), 2, g, slots=t(1, dtype=torch.int32))),
        (TypeError, lambda: ops.linear_attention(t(1, 4, 128), t(1, 4, 128), t(1, 4, 128), 2, g, state=t(1, 2, 64, 64))),
        (ValueError, lambda: ops.linear_attention(t(4, 128), t(4, 128), t(4, 128), 2, g, seg_start=t(2, dtype=torch.int32))),
        (TypeError, lambda: ops.linear_attention(t(4, 128), t(4, 128), t(4, 128), 2, g, seg_start=t(2, dtype=torch.int64), max_seg_rows=4)),
        (KatzHipError, lambda: ops.linear_attention(t(1, 4, 96), t(1, 4, 96), t(1, 4, 96), 2, g)),
        (KatzHipError, lambda: ops.linear_attention(t(1, 4, 132)[..., :128], t(1, 4, 128), t(1, 4, 128), 2, g)),
        (ValueError, lambda: ops.linear_attention(t(2, 4, 128), t(2, 4, 128), t(2, 4, 128), 2, g, out=t(1, 4, 128).expand(2, 4, 128))),
        (ValueError, lambda: ops.linear_attention_step(t(2, 128), t(2, 128), t(2, 128), 2, g, t(3, 2, 64, 64, dtype=f))),
        (TypeError, lambda: ops.linear_attention_step(t(2, 128), t(2, 128), t(2, 128), 2, g, t(3, 2, 64, 64, dtype=f), slots=t(2, dtype=torch.int64))),
    ]
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            pytest.fail(f"call {i} was not refused")


def test_launches_that_would_be_too_large(lib):
    """More threads than a launch takes; scales and zero points at addresses that whole rows cannot have."""
    norm = lambda M, D: lib.kh_block_norm(16, 16, None, 1, None, None, None, None, 16, 16, M, D, 1.0, 1e-6, 0, 0, 0, None)      # noqa: E731
    assert norm(1 << 26, 64) == -4 and norm(1 << 24, 4096) == -4 and norm(1 << 22, 32768) == -4
    linear = lambda s=16, z=None: lib.kh_w4_linear(16, 16, s, z, None, None, None, None, None, 16, None, 2, 8, 64, 0, 64, 0, None)      # noqa: E731
    assert linear(s=20) == -3 and linear(z=18) == -3


def test_wide_linears(lib):
    """More rank columns than the adapters' other entry points take, up to a limit of its own."""
    size = lib.kh_w4_linear_wide_workspace_bytes
    assert size(1, 64, 160) > 0 and size(40, 1280, 160) >= 6 * 40 * 160 and size(1, 64, 150) == -1 and size(1, 64, 65568) == -1 and size(1, 64, 32) == 0
    wide = lambda R, ws=16, g=64: lib.kh_w4_linear_wide(16, 16, 16, None, None, 16, 16, 16, None, 16, ws, 2, 8, 64, R, g, 0, None)      # noqa: E731
    assert wide(65568) == -4 and wide(150) == -2 and wide(160, ws=None) == -1 and wide(160, g=48) == -2


def test_w4_linear_refuses_workspaces_and_scales_off_their_alignment(lib):
    """The ranks' products are read from the workspace 16 bytes at a time, column scales as floats."""
    for f in (lib.kh_w4_linear, lib.kh_w4_linear_wide):
        call = lambda ws=16, c=16, M=2, K=8192, R=64: f(16, 16, 16, None, None, 16, 16, c, None, 16, ws, M, 8, K, R, 64, 0, None)      # noqa: E731
        assert call(ws=20) == -3 and call(ws=24, M=700) == -3 and call(c=18) == -3 and call(ws=None, c=18, K=64) == -3


# A HIP runtime's calls for launches, of which the fail_at-th fails as one does: an error that the next hipGetLastError returns and clears.
LAUNCHES = """
typedef struct { unsigned x, y, z; } dim3;
int launches, fail_at;
static int last;
int __hipPushCallConfiguration(dim3 g, dim3 b, unsigned long lds, void* s) { return 0; }
int __hipPopCallConfiguration(dim3* g, dim3* b, unsigned long* lds, void** s) { dim3 one = {1, 1, 1}; *g = *b = one; *lds = 0; *s = 0; return 0; }
int hipLaunchKernel(const void* f, dim3 g, dim3 b, void** args, unsigned long lds, void* s) { if (++launches == fail_at) last = 719; return launches == fail_at ? 719 : 0; }
int hipGetLastError(void) { int e = last; last = 0; return e; }
int hipGetDevice(int* d) { *d = 0; return 0; }
int hipFuncSetAttribute(const void* f, int a, int v) { return 0; }
"""
CALLS = """
import ctypes, sys
fake = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
from katz_amd import _lib
lib = _lib.load()
calls = {"prompt": (3, lambda: lib.kh_linear_attention_bf16(16, 16, 16, 16, 16, None, 16, None, 1, None, 0, 16, 1, 2, 2, 4096, 64, 64, *[128] * 4, *[0] * 4, 0.1, None)),
         "linear": (2, lambda: lib.kh_w4_linear(16, 16, 16, None, None, 16, 16, 16, None, 16, 16, 2, 8, 8192, 64, 64, 0, None))}
count, failing = ctypes.c_int.in_dll(fake, "launches"), ctypes.c_int.in_dll(fake, "fail_at")
for name, (n, call) in calls.items():
    for at in range(n + 1):
        count.value, failing.value = 0, at
        rc = call()
        print(name, n, at, rc, count.value)
"""


def test_a_launch_that_fails_ends_its_call(lib, tmp_path):
    """Whichever launch of a call fails, the call returns that error and launches nothing behind it, which would read what the failed one has not written."""
    if not shutil.which("gcc"):
        pytest.skip("no gcc")
    (tmp_path / "launches.c").write_text(LAUNCHES)
    subprocess.run(["gcc", "-shared", "-fPIC", "-w", "-o", str(tmp_path / "launches.so"), str(tmp_path / "launches.c")], check=True)
    run = subprocess.run([sys.executable, "-c", CALLS, str(tmp_path / "launches.so")], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stderr
    lines = [line.split() for line in run.stdout.splitlines()]
    assert len(lines) == 7
    for name, n, at, rc, count in lines:
        assert (rc, count) == (("0", n) if at == "0" else ("719", at)), (name, at, rc, count)


def test_linear_attention_plans_for_as_many_workgroups_as_run_at_once(lib):
    """Chunks of few long sequences fill the CUs once, whatever the shape of a head: the fastest of the counts that were measured."""
    def chunks(B, H, T, dk, dv):
        n = lib.kh_linear_attention_workspace_bytes(B, H, T, B * T, dk, dv)
        one = H * dk * dv * 8 + 16                         # two states of every head and the chunk's place
        assert n % one == 0
        return n // one

    assert chunks(1, 16, 16384, 64, 128) == 16 and chunks(2, 20, 4096, 64, 128) == 12
    assert chunks(1, 16, 16384, 128, 64) == 16 and chunks(2, 20, 4096, 128, 64) == 12
    assert chunks(1, 16, 16384, 128, 128) == 16 and chunks(1, 16, 16384, 64, 64) == 32         # (two workgroups to a CU)
    assert chunks(16, 16, 1024, 128, 128) == chunks(4, 40, 512, 64, 64) == 0                    # whole sequences
