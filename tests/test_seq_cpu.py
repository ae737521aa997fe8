"""CPU checks of the sequence operators: the exported C entry points, their argument validation (which returns before any
CUDA call; the fake pointers are never dereferenced), the oracle against closed forms, and the public names."""

from __future__ import annotations

import ctypes
import math
import re
from pathlib import Path

import pytest
import torch

from oracle import seq64

ROOT = Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "cufkb_seq.h"

SUCCESS, INVALID_DTYPE, NULL_POINTER, POINT_COUNT, TOO_MANY_STEPS, SHAPE_LIMITS, BAD_STRIDE, MISALIGNED, INVALID_VALUE, CUDA, WORKSPACE, UNSUPPORTED = range(12)
F32, F64, F16, BF16 = range(4)
vp, i64, ci = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int


class ConvParams(ctypes.Structure):
    _fields_ = [
        ("dtype", ci), ("taps", ci), ("silu", ci), ("rows", i64), ("chains", i64), ("width", i64), ("chain_points", vp), ("x", vp), ("x_stride", i64),
        ("weight", vp), ("bias", vp), ("initial_state", vp), ("y", vp), ("final_state", vp), ("grad_y", vp), ("grad_y_stride", i64),
        ("grad_final_state", vp), ("grad_x", vp), ("grad_weight", vp), ("grad_bias", vp), ("grad_initial_state", vp), ("workspace", vp),
        ("workspace_bytes", ctypes.c_size_t),
    ]


class ScanParams(ctypes.Structure):
    _fields_ = [
        ("dtype", ci), ("softplus", ci), ("rows", i64), ("chains", i64), ("width", i64), ("groups", i64), ("states", i64), ("chain_points", vp), ("x", vp),
        ("delta", vp), ("z", vp), ("x_stride", i64), ("delta_stride", i64), ("z_stride", i64), ("A", vp), ("B", vp), ("C", vp), ("B_stride", i64),
        ("B_group_stride", i64), ("C_stride", i64), ("C_group_stride", i64), ("D", vp), ("delta_bias", vp), ("initial_state", vp), ("y", vp),
        ("final_state", vp), ("checkpoints", vp), ("grad_y", vp), ("grad_y_stride", i64), ("grad_final_state", vp), ("grad_x", vp), ("grad_delta", vp),
        ("grad_z", vp), ("grad_B", vp), ("grad_C", vp), ("grad_A", vp), ("grad_D", vp), ("grad_delta_bias", vp), ("grad_initial_state", vp),
        ("workspace", vp), ("workspace_bytes", ctypes.c_size_t),
    ]


class GradArray(ctypes.Structure):
    _fields_ = [("grad", vp), ("out", vp), ("count", i64), ("dtype", ci)]


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(str(ROOT / "cufk_b200" / "libcufkb.so"))
    lib.cufkb_conv_step.argtypes = [ci, vp, i64, vp, vp, vp, vp, i64, i64, ci, ci, vp]
    lib.cufkb_token_logprobs.argtypes = [ci, vp, i64, vp, vp, vp, vp, vp, vp, i64, i64, ci, vp]
    lib.cufkb_token_logprobs_backward.argtypes = [ci, vp, i64, vp, vp, vp, vp, vp, vp, i64, i64, vp]
    lib.cufkb_clip_gradients.argtypes = [vp, i64, ctypes.c_double, ctypes.c_double, vp, ci, vp, ctypes.c_size_t, vp]
    lib.cufkb_clip_workspace_bytes.argtypes = [vp, i64, vp]
    lib.cufkb_seq_status_string.restype = ctypes.c_char_p
    return lib


def test_library_exports_every_declared_symbol(lib):
    names = set(re.findall(r"^\s*CUFKB_API\s+(?:const\s+)?\w+\*?\s+\*?(cufkb_\w+)\s*\(", HEADER.read_text(), flags=re.M))
    assert {"cufkb_conv_forward", "cufkb_scan_backward", "cufkb_token_logprobs", "cufkb_clip_gradients"} <= names
    for name in names:
        assert hasattr(lib, name), name


def test_public_names():
    import cufk_b200 as cufk

    for name in cufk.seq.__all__:
        assert hasattr(cufk.seq, name)


def conv(**kw):
    base = dict(dtype=F32, taps=4, silu=1, rows=10, chains=2, width=8, x=64, x_stride=8, weight=64, y=64)
    base.update(kw)
    return ConvParams(**base)


@pytest.mark.parametrize(
    "change, status",
    [
        (dict(dtype=9), INVALID_DTYPE), (dict(dtype=F64), UNSUPPORTED), (dict(taps=1), INVALID_VALUE), (dict(taps=5), INVALID_VALUE),
        (dict(rows=-1), SHAPE_LIMITS), (dict(rows=9), SHAPE_LIMITS), (dict(chains=0), SHAPE_LIMITS), (dict(width=-2), SHAPE_LIMITS),
        (dict(x=None), NULL_POINTER), (dict(y=None), NULL_POINTER), (dict(weight=None), NULL_POINTER), (dict(x=66), MISALIGNED),
        (dict(weight=66), MISALIGNED), (dict(chain_points=12), MISALIGNED), (dict(x_stride=-8), BAD_STRIDE), (dict(width=0, x=None, y=None), SUCCESS),
        (dict(rows=0, x=None, y=None), SUCCESS),
    ],
)
def test_conv_forward_validation(lib, change, status):
    assert lib.cufkb_conv_forward(ctypes.byref(conv(**change)), None) == status


@pytest.mark.parametrize(
    "change, status",
    [
        (dict(grad_y=None), NULL_POINTER), (dict(grad_weight=64), NULL_POINTER), (dict(grad_weight=64, grad_bias=64), WORKSPACE),
        (dict(grad_weight=64, grad_bias=64, workspace=64, workspace_bytes=8), WORKSPACE), (dict(grad_y_stride=-1), BAD_STRIDE), (dict(grad_x=65), MISALIGNED),
    ],
)
def test_conv_backward_validation(lib, change, status):
    base = dict(grad_y=64, grad_y_stride=8, grad_x=64)
    base.update(change)
    assert lib.cufkb_conv_backward(ctypes.byref(conv(**base)), None) == status


def scan(**kw):
    base = dict(dtype=F32, softplus=1, rows=10, chains=2, width=8, groups=1, states=16, x=64, delta=64, x_stride=8, delta_stride=8, A=64, B=64, C=64, B_stride=16, C_stride=16, y=64)
    base.update(kw)
    return ScanParams(**base)


@pytest.mark.parametrize(
    "change, status",
    [
        (dict(dtype=9), INVALID_DTYPE), (dict(dtype=F64), UNSUPPORTED), (dict(states=0), INVALID_VALUE), (dict(states=65), INVALID_VALUE),
        (dict(groups=0), INVALID_VALUE), (dict(groups=3), INVALID_VALUE), (dict(rows=11), SHAPE_LIMITS), (dict(chains=-1), SHAPE_LIMITS),
        (dict(B_stride=-1), BAD_STRIDE), (dict(x_stride=2**24 + 1), BAD_STRIDE), (dict(rows=2**36, chains=1, width=2**20, x_stride=2**20), SHAPE_LIMITS), (dict(A=None), NULL_POINTER), (dict(B=None), NULL_POINTER), (dict(y=None), NULL_POINTER), (dict(z=65), MISALIGNED),
        (dict(checkpoints=8), MISALIGNED), (dict(rows=100000, chains=1), WORKSPACE), (dict(width=0), SUCCESS),
    ],
)
def test_scan_forward_validation(lib, change, status):
    assert lib.cufkb_scan_forward(ctypes.byref(scan(**change)), None) == status


@pytest.mark.parametrize(
    "change, status",
    [
        (dict(grad_y=None), NULL_POINTER), (dict(grad_A=None), NULL_POINTER), (dict(z=64), NULL_POINTER), (dict(checkpoints=None), WORKSPACE),
        (dict(workspace_bytes=16), WORKSPACE),
    ],
)
def test_scan_backward_validation(lib, change, status):
    base = dict(grad_y=64, grad_y_stride=8, grad_x=64, grad_delta=64, grad_A=64, grad_B=64, grad_C=64, checkpoints=64, workspace=64, workspace_bytes=1 << 30)
    base.update(change)
    assert lib.cufkb_scan_backward(ctypes.byref(scan(**base)), None) == status


def test_step_validation(lib):
    assert lib.cufkb_scan_step(ctypes.byref(scan(final_state=None)), None) == NULL_POINTER
    assert lib.cufkb_scan_step(ctypes.byref(scan(chains=0, x=None)), None) == SUCCESS
    assert lib.cufkb_conv_step(F32, 64, 8, None, 64, None, 64, 2, 8, 4, 1, None) == NULL_POINTER
    assert lib.cufkb_conv_step(F32, 64, 8, 64, 64, None, 64, 2, 8, 6, 1, None) == INVALID_VALUE
    assert lib.cufkb_conv_step(F64, 64, 8, 64, 64, None, 64, 2, 8, 4, 1, None) == UNSUPPORTED
    assert lib.cufkb_conv_step(F32, 64, 8, 64, 64, None, 64, 0, 8, 4, 1, None) == SUCCESS


def test_scan_sizes(lib):
    size = ctypes.c_size_t()
    assert lib.cufkb_scan_checkpoint_bytes(ctypes.byref(scan(rows=160, chains=1)), ctypes.byref(size)) == SUCCESS
    assert size.value >= 10 * 8 * 16 * 4
    assert lib.cufkb_scan_workspace_bytes(ctypes.byref(scan()), 0, ctypes.byref(size)) == SUCCESS and size.value == 0
    assert lib.cufkb_scan_workspace_bytes(ctypes.byref(scan()), 1, ctypes.byref(size)) == SUCCESS and size.value > 0
    assert lib.cufkb_scan_workspace_bytes(None, 1, ctypes.byref(size)) == NULL_POINTER


def logprobs(lib, dtype=F32, logits=64, stride=8, tokens=64, logp=64, entropy=64, log_sum=64, top_logp=64, top_tokens=64, rows=2, n=8, top=2):
    return lib.cufkb_token_logprobs(dtype, logits, stride, tokens, logp, entropy, log_sum, top_logp, top_tokens, rows, n, top, None)


def test_logprobs_validation(lib):
    assert logprobs(lib, dtype=F64) == UNSUPPORTED
    assert logprobs(lib, n=0) == SHAPE_LIMITS
    assert logprobs(lib, rows=-1) == SHAPE_LIMITS
    assert logprobs(lib, top=33, n=64) == INVALID_VALUE
    assert logprobs(lib, top=9) == INVALID_VALUE
    assert logprobs(lib, top=-1) == INVALID_VALUE
    assert logprobs(lib, stride=-8) == BAD_STRIDE
    assert logprobs(lib, logits=66) == MISALIGNED
    assert logprobs(lib, tokens=68) == MISALIGNED
    assert logprobs(lib, top_tokens=None) == NULL_POINTER
    assert logprobs(lib, tokens=None) == NULL_POINTER
    assert logprobs(lib, rows=0, logits=None) == SUCCESS
    assert lib.cufkb_token_logprobs_backward(F32, 64, 8, 64, 64, 64, 64, 64, None, 2, 8, None) == NULL_POINTER
    assert lib.cufkb_token_logprobs_backward(F32, 64, 8, 64, 64, 64, None, None, 65, 2, 8, None) == MISALIGNED


def test_clip_validation(lib):
    size = ctypes.c_size_t()

    def call(array, count=1, max_norm=1.0, eps=1e-6, norm=64, dtype=F32, ws=64, ws_bytes=1 << 20):
        return lib.cufkb_clip_gradients(ctypes.byref(array) if array is not None else None, count, max_norm, eps, norm, dtype, ws, ws_bytes, None)

    good = GradArray(64, 64, 10, F32)
    assert call(GradArray(64, 64, 10, 7)) == INVALID_DTYPE
    assert call(GradArray(None, 64, 10, F32)) == NULL_POINTER
    assert call(GradArray(66, 64, 10, F32)) == MISALIGNED
    assert call(GradArray(64, 64, -1, F32)) == SHAPE_LIMITS
    assert call(GradArray(64, 64, 2**34 + 1, F32)) == SHAPE_LIMITS
    assert call(None) == NULL_POINTER
    assert call(good, max_norm=-1.0) == INVALID_VALUE
    assert call(good, max_norm=math.nan) == INVALID_VALUE
    assert call(good, norm=None) == NULL_POINTER
    assert call(good, dtype=F16) == UNSUPPORTED
    assert call(good, ws_bytes=8) == WORKSPACE
    assert call(good, ws=68) == MISALIGNED
    assert lib.cufkb_clip_workspace_bytes(ctypes.byref(good), 1, ctypes.byref(size)) == SUCCESS and size.value > 0


def test_status_strings(lib):
    for status in range(13):
        assert lib.cufkb_seq_status_string(status)


def test_oracle_scan_against_closed_form():
    # constant inputs: h_t = u B (1 - a^t) / (1 - a)
    rows, dt = 9, 0.3
    x = torch.full((rows, 1), 2.0, dtype=torch.float64)
    delta = torch.full((rows, 1), dt, dtype=torch.float64)
    A = torch.tensor([[-0.5]], dtype=torch.float64)
    one = torch.ones(rows, 1, 1, dtype=torch.float64)
    y, state = seq64.selective_scan(x, delta, A, one, one, use_softplus=False)
    a = math.exp(dt * -0.5)
    want = torch.tensor([[dt * 2.0 * (1 - a**t) / (1 - a)] for t in range(1, rows + 1)], dtype=torch.float64)
    assert torch.allclose(y, want, rtol=1e-12)
    assert torch.allclose(state[0], want[-1:], rtol=1e-12)


def test_oracle_conv_against_torch():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(12, 5, generator=g, dtype=torch.float64)
    w = torch.randn(5, 4, generator=g, dtype=torch.float64)
    y, state = seq64.short_conv(x, w, use_silu=False)
    want = torch.nn.functional.conv1d(torch.nn.functional.pad(x.t()[None], (3, 0)), w[:, None], groups=5)[0].t()
    assert torch.allclose(y, want, rtol=1e-12, atol=1e-13)
    assert torch.equal(state[0], x[-3:])


def test_oracle_logprobs_against_torch():
    g = torch.Generator().manual_seed(1)
    logits = torch.randn(6, 11, generator=g, dtype=torch.float64)
    tokens = torch.tensor([0, 10, 3, -1, 11, 5])
    logp, entropy, top, ids = seq64.token_logprobs(logits, tokens, 3)
    dist = torch.distributions.Categorical(logits=logits)
    assert torch.allclose(entropy, dist.entropy())
    assert torch.allclose(logp[[0, 1, 2, 5]], dist.log_prob(tokens.clamp(0, 10))[[0, 1, 2, 5]])
    assert logp[3] == 0 and torch.isnan(logp[4])
    assert torch.equal(ids, logits.topk(3).indices)


def test_refusals_without_a_gpu():
    from cufk_b200 import seq

    x, w = torch.zeros(4, 8), torch.zeros(8, 4)
    with pytest.raises(RuntimeError, match="x must be CUDA"):
        seq.short_conv(x, w)
    with pytest.raises(RuntimeError, match="x must be CUDA"):
        seq.selective_scan(x, x, torch.zeros(8, 16), torch.zeros(4, 16), torch.zeros(4, 16))
    with pytest.raises(RuntimeError, match="logits must be CUDA"):
        seq.token_logprobs(x, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="must be CUDA"):
        seq.clip_gradients([x], 1.0)
    with pytest.raises(RuntimeError, match="at least one gradient"):
        seq.clip_gradients([], 1.0)
    with pytest.raises(RuntimeError, match="must not be negative"):
        seq.clip_gradients([x], -1.0)


def test_dependent_kernels_promise_nothing_about_memory():
    # a kernel that starts before the one in front has ended reads nothing that it declares unchanging: what that one writes changes
    # while this one runs, and a restrict pointer would allow its reads to be made before the wait
    for name in ("conv_kernels.cuh", "scan_kernels.cuh"):
        source = (ROOT / "cufk_b200" / "csrc" / name).read_text()
        kernels = re.split(r"(?=__global__ )", source)[1:]
        waiting = [k for k in kernels if "wait_for_previous()" in k]
        assert waiting
        for kernel in waiting:
            assert "__restrict__" not in kernel.split("{")[0]


def test_clip_refuses_shared_memory(lib):
    def call(*arrays):
        list_of = (GradArray * len(arrays))(*[GradArray(*a) for a in arrays])
        return lib.cufkb_clip_gradients(list_of, len(arrays), 1.0, 1e-6, 64, F32, 64, 1 << 30, None)

    refused = [
        [(4096, 4096, 10, F32), (4132, 4132, 10, F32)],                              # in place, one element in common
        [(4132, 4132, 10, F32), (4096, 4096, 10, F32)],
        [(4096, 4096, 10, F32), (4096, 4096, 9, F32)],                               # the same start
        [(4096, 4096, 10, F32), (4096, 4096, 10, BF16)],                             # the same memory as another type
        [(4096, 8192, 10, F32), (4200, 8228, 10, F32)],                              # results in common
        [(4096, 8192, 10, F32), (8192, 12288, 10, F32)],                             # a result over another's gradient
        [(8192, 12288, 10, F32), (4096, 8192, 10, F32)],
        [(4096, 4100, 10, F32)],                                                     # over a part of its own gradient
        [(4096, 4096, 10, F32), (4096, 8192, 10, F32)],                              # written and read again
        [(4096, 8192, 10, F32), (4096, 4096, 10, F32)],
        [(4096, 4096, 1000, F32), (4100, 4100, 1, F32), (4096, 4096, 1000, F32)],    # in the middle of a repeated one
        [(4096, 4096, 10, F32), (4096, 4096, 10, F32), (4120, 4120, 1, F32)],
    ]
    for arrays in refused:
        assert call(*arrays) == INVALID_VALUE, arrays


def test_dependent_kernels_declare_no_input_unchanging():
    # the same for the kernels of the reconstruction: const with restrict is what allows a read before the wait
    found = 0
    for path in (ROOT / "cufk_b200" / "csrc").glob("*.cuh"):
        for kernel in re.split(r"(?=__global__ )", path.read_text())[1:]:
            if "enter_after_previous_grid()" in kernel or "wait_for_previous()" in kernel:
                found += 1
                assert not re.search(r"const [^,()]*\* __restrict__", kernel.split("{")[0]), path.name
    assert found >= 10
