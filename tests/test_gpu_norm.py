"""The residual norm on the GPU against the formula in 64 bits.

Tolerances.  u = 2^-24 is the relative error of one FP32 rounding.  A thread adds at most 32
squares, a warp 5 partial sums, a block 32: all terms are positive, so the mean is within 70 u,
its square root within 35 u; rsqrtf (2 ulp), the sum, and two products add 7 u.  48 u < 2^-18
covers y.  The results' own roundings: 2^-8 relative in BF16, 2^-4 in E4M3 (2^-10 absolute below
its smallest normal value), u for an FP32 residual.
"""

from __future__ import annotations

import pytest
import torch

from b200moe import add_rms_norm, add_rms_norm_fp8, dequantize_rows_fp8, quantize_rows_fp8

pytestmark = pytest.mark.gpu

FP32 = 2.0 ** -18
U = 2.0 ** -24


def _inputs(device, rows, hidden, residual, weight, seed=5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, hidden, generator=g).bfloat16().to(device)
    r = None if residual is None else (3 * torch.randn(rows, hidden, generator=g)).to(residual).to(device)
    w = (1 + 0.2 * torch.randn(hidden, generator=g)).to(weight).to(device)
    return x, r, w


def _formula(x, r, w, eps):
    s = x.double().cpu() + (0 if r is None else r.double().cpu())
    return s, s / (s.square().mean(-1, keepdim=True) + eps).sqrt() * w.double().cpu()


def _near(got, want, rel, absolute=0.0):
    got = got.double().cpu()
    off = (got - want).abs() - (rel * want.abs() + absolute)
    assert got.shape == want.shape and bool((off <= 0).all()), float(off.max())


def _check_residual(got, s, r):
    _near(got, s, 2.0 ** -8 + U if r.dtype is torch.bfloat16 else U)


SHAPES = [(1, 8), (3, 64), (1, 200), (64, 2880), (257, 72), (2, 4096), (5, 8200), (3, 16384),
          (1, 32768), (1000, 16)]
TYPES = [(None, torch.bfloat16), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
         (torch.float32, torch.bfloat16), (torch.float32, torch.float32), (None, torch.float32)]


@pytest.mark.parametrize("rows, hidden", SHAPES)
@pytest.mark.parametrize("residual, weight", TYPES)
def test_bf16_rows(cuda_device, rows, hidden, residual, weight) -> None:
    x, r, w = _inputs(cuda_device, rows, hidden, residual, weight)
    out, kept = add_rms_norm(x, r, w, eps=1e-5)
    s, y = _formula(x, r, w, 1e-5)
    _near(out, y, 2.0 ** -8 + FP32)
    assert out.dtype is torch.bfloat16
    if r is None:
        assert kept is x
    else:
        assert kept.dtype is r.dtype
        _check_residual(kept, s, r)


@pytest.mark.parametrize("rows, hidden", [s for s in SHAPES if s[1] % 16 == 0])
@pytest.mark.parametrize("residual, weight", TYPES)
def test_e4m3_rows(cuda_device, rows, hidden, residual, weight) -> None:
    x, r, w = _inputs(cuda_device, rows, hidden, residual, weight)
    codes, scale, kept = add_rms_norm_fp8(x, r, w)
    s, y = _formula(x, r, w, 1e-6)
    want = y.abs().amax(-1) / 448.0
    _near(scale, want, FP32)
    quotient = y / want[:, None]
    _near(codes.view(torch.float8_e4m3fn).float(), quotient, 2.0 ** -4 + 3 * FP32, 2.0 ** -10)
    assert codes.dtype is torch.uint8 and scale.shape == (rows,)
    if r is not None:
        _check_residual(kept, s, r)


def test_codes_follow_the_row_quantiser(cuda_device) -> None:
    """On rows that BF16 holds exactly, norm and quantiser in one give what the quantiser gives:
    |s| = 1 throughout and eps = 0 make y = +-w, w powers of two."""

    g = torch.Generator().manual_seed(1)
    x = (torch.randint(0, 2, (7, 256), generator=g) * 2 - 1).bfloat16().to(cuda_device)
    w = (2.0 ** torch.randint(-6, 4, (256,), generator=g)).bfloat16().to(cuda_device)
    codes, scale, _ = add_rms_norm_fp8(x, None, w, eps=0.0)
    q, qs = quantize_rows_fp8((x * w).contiguous())
    assert torch.equal(codes, q) and torch.equal(scale, qs)
    back = dequantize_rows_fp8(codes, scale)
    _near(back, (x * w).double().cpu(), 2.0 ** -4 + 2.0 ** -8, 2.0 ** -10 * float(scale.max()))


def test_leading_dimensions_and_no_rows(cuda_device) -> None:
    x, r, w = _inputs(cuda_device, 6, 128, torch.float32, torch.bfloat16)
    flat, kept = add_rms_norm(x, r, w)
    out, kept3 = add_rms_norm(x.view(2, 3, 128), r.view(2, 3, 128), w)
    assert torch.equal(out.view(6, 128), flat) and torch.equal(kept3.view(6, 128), kept)
    one, _ = add_rms_norm(x[0], r[0], w)
    assert one.shape == (128,) and torch.equal(one, flat[0])
    codes, scale, _ = add_rms_norm_fp8(x[0], r[0], w)
    assert codes.shape == (128,) and scale.shape == ()
    out, kept = add_rms_norm(x[:0], r[:0], w)
    assert out.shape == kept.shape == (0, 128)
    codes, scale, _ = add_rms_norm_fp8(x[:0], r[:0], w)
    assert codes.shape == (0, 128) and scale.shape == (0,)


def test_rows_of_zeros_and_non_finite_values(cuda_device) -> None:
    x, r, w = _inputs(cuda_device, 5, 512, torch.bfloat16, torch.bfloat16)
    x[1] = 0
    r[1] = 0
    x[2, 17] = float("inf")
    x[3, 5] = float("nan")
    out, kept = add_rms_norm(x, r, w)
    codes, scale, _ = add_rms_norm_fp8(x, r, w)
    assert bool((out[1] == 0).all()) and bool((codes[1] == 0).all()) and float(scale[1]) == 1.0
    # 1 / sqrt(inf) = 0: the infinite element becomes NaN, the others zero
    assert bool(out[2, 17].isnan()) and int(out[2].isnan().sum()) == 1
    assert bool((out[2].nan_to_num(0.0) == 0).all())
    assert bool(out[3].isnan().all())
    assert float(kept[2, 17]) == float("inf") and bool(kept[3, 5].isnan())
    s, y = _formula(x[[0, 4]], r[[0, 4]], w, 1e-6)  # the rows beside them are untouched
    _near(out[[0, 4]], y, 2.0 ** -8 + FP32)


@pytest.mark.parametrize("fp8", [False, True])
def test_results_in_the_callers_tensors(cuda_device, fp8) -> None:
    x, r, w = _inputs(cuda_device, 9, 1024, torch.bfloat16, torch.float32)
    if fp8:
        want = add_rms_norm_fp8(x, r, w)
        bufs = [torch.empty_like(t) for t in want]
        got = add_rms_norm_fp8(x, r, w, out=bufs[0], scale_out=bufs[1], residual_out=bufs[2])
    else:
        want = add_rms_norm(x, r, w)
        bufs = [torch.empty_like(t) for t in want]
        got = add_rms_norm(x, r, w, out=bufs[0], residual_out=bufs[1])
    assert all(a is b and torch.equal(a, c) for a, b, c in zip(got, bufs, want))


def test_in_place(cuda_device) -> None:
    x, r, w = _inputs(cuda_device, 33, 2880, torch.bfloat16, torch.bfloat16)
    want, kept = add_rms_norm(x, r, w)
    a, b = x.clone(), r.clone()
    add_rms_norm(a, b, w, out=a, residual_out=b)      # each over its own input
    assert torch.equal(a, want) and torch.equal(b, kept)
    a, b = x.clone(), r.clone()
    add_rms_norm(a, b, w, out=b, residual_out=a)      # crosswise
    assert torch.equal(b, want) and torch.equal(a, kept)


def test_overlaps_and_wrong_buffers_are_refused(cuda_device) -> None:
    x, r, w = _inputs(cuda_device, 4, 64, torch.bfloat16, torch.bfloat16)
    pool = torch.zeros(5 * 64, dtype=torch.bfloat16, device=cuda_device)
    first, shifted = pool[:256].view(4, 64), pool[64:].view(4, 64)
    first.copy_(x)
    with pytest.raises(ValueError, match="overlap"):
        add_rms_norm(first, r, w, out=shifted)
    with pytest.raises(ValueError, match="overlap"):
        add_rms_norm(x, r, w, out=first, residual_out=first)
    with pytest.raises(ValueError, match="overlap the weight"):
        add_rms_norm(x[0], None, w, out=w)
    with pytest.raises(ValueError, match="residual_out"):
        add_rms_norm(x, r, w, residual_out=r.float())
    with pytest.raises(ValueError, match="needs a residual"):
        add_rms_norm(x, None, w, residual_out=torch.empty_like(x))
    with pytest.raises(ValueError, match="out must be"):
        add_rms_norm(x, r, w, out=torch.empty(4, 64, device=cuda_device))
    with pytest.raises(ValueError, match="out must be"):
        add_rms_norm(x, r, w, out=torch.empty(4, 64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="scale_out must be"):
        add_rms_norm_fp8(x, r, w, scale_out=torch.empty(5, device=cuda_device))
    with pytest.raises(ValueError, match="same device"):
        add_rms_norm(x, r.cpu(), w)
    with pytest.raises(ValueError, match="16-byte"):  # rows that start between 16-byte boundaries
        add_rms_norm(pool[1:257].view(4, 64), r, w)


def test_on_another_stream_and_in_a_graph(cuda_device) -> None:
    x, r, w = _inputs(cuda_device, 64, 4096, torch.float32, torch.bfloat16)
    want, kept = add_rms_norm(x, r, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, kept2 = add_rms_norm(x, r, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(kept2, kept)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, kept2 = add_rms_norm(x, r, w)
        codes, scale, _ = add_rms_norm_fp8(x, r, w)
    x2, r2, _ = _inputs(cuda_device, 64, 4096, torch.float32, torch.bfloat16, seed=6)
    x.copy_(x2)
    r.copy_(r2)
    graph.replay()
    want, kept = add_rms_norm(x2, r2, w)
    wcodes, wscale, _ = add_rms_norm_fp8(x2, r2, w)
    assert torch.equal(got, want) and torch.equal(kept2, kept)
    assert torch.equal(codes, wcodes) and torch.equal(scale, wscale)
