"""8-bit activation checkpoints: the copy is `mxfp8_quantize`'s, and it comes back as the values that its codes stand for."""

import pytest
import torch

from miles_amd import launch
from miles_amd.kernels.quant.act_checkpoint import ActCheckpoint, checkpoint_activation
from miles_amd.utils.mxfp8 import mxfp8_dequantize, mxfp8_quantize
from tests.operator_checks import f64, restored64, within

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _x(shape, dtype, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(3 * torch.randn((*shape[:-1], 1), generator=g)) * scale
    return x.to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 32), (32,), (3, 5, 64), (257, 96), (1031, 2560), (0, 64)])
def test_round_trip(shape, dtype):
    x = _x(shape, dtype, 1) if 0 not in shape else torch.empty(shape, dtype=dtype, device=DEV)
    kept = checkpoint_activation(x)
    q, s = mxfp8_quantize(x)
    assert torch.equal(kept.codes.view(torch.uint8), q.view(torch.uint8)) and torch.equal(kept.scales, s)
    assert kept.shape == x.shape and kept.dtype == dtype and kept.nbytes == q.nbytes + s.nbytes
    want = restored64(kept.codes, kept.scales)
    for out in TYPES:
        got = kept.restore(out)
        expect = want.clamp(-65504, 65504) if out == torch.float16 else want
        assert got.dtype == out and torch.equal(f64(got), f64(expect.to(out)))
    assert kept.restore().dtype == dtype
    # half a step of e4m3 of the value, or of the smallest step of its group (2^-9 of the scale)
    if x.numel():
        scale = torch.pow(torch.tensor(2.0, dtype=torch.float64), kept.scales.cpu().double() - 127).repeat_interleave(32, -1).to(DEV)
        assert ((want - f64(x)).abs() <= 2.0**-4 * f64(x).abs() + 2.0**-10 * scale).all()


@pytest.mark.parametrize("out", TYPES)
def test_every_code_under_every_scale(out):
    codes = torch.arange(256, dtype=torch.uint8, device=DEV).repeat(255, 1)
    scales = torch.arange(255, dtype=torch.uint8, device=DEV).unsqueeze(1).expand(255, 8).contiguous()
    got = mxfp8_dequantize(codes.view(torch.float8_e4m3fn), scales, out).cpu()
    want = restored64(codes.view(torch.float8_e4m3fn).cpu(), scales.cpu())
    if out == torch.float16:
        want = want.clamp(-65504, 65504)
    want = want.to(out) if out != torch.float32 else want.float()
    assert torch.equal(got.isnan(), want.isnan())
    fine = ~want.isnan()
    assert torch.equal(got[fine], want[fine])


def test_special_values():
    x = torch.zeros(4, 64, device=DEV)
    x[0, 3], x[1, 40], x[2, :32] = float("inf"), float("nan"), 1e-42
    x[0, 4], x[1, 41] = 3.0, -7.0
    kept = checkpoint_activation(x)
    back = kept.restore()
    assert back[1, 40].isnan() and back[1, 41] == -7 and back[1].isnan().sum() == 1
    assert back[0, 3] > 1e38 and (back[3] == 0).all() and (back[2] == 0).all()


def test_strided_and_misaligned_inputs():
    big = _x((70, 200), torch.bfloat16, 3)
    for x in (big[:, 8:168], big[3:67].t()[:, :64], big[:, 3:163]):
        kept = checkpoint_activation(x)
        q, s = mxfp8_quantize(x.contiguous())
        assert torch.equal(kept.codes.view(torch.uint8), q.view(torch.uint8)) and torch.equal(kept.scales, s)
    codes = torch.zeros(64 * 64 + 1, dtype=torch.uint8, device=DEV)[1:].view(64, 64)
    codes.copy_(torch.arange(64, dtype=torch.uint8, device=DEV))
    scales = torch.full((64, 2), 127, dtype=torch.uint8, device=DEV)
    assert torch.equal(mxfp8_dequantize(codes, scales, torch.float32), codes.view(torch.float8_e4m3fn).float())


def test_made_at_once_inside_a_deferred_block():
    x = _x((64, 128), torch.bfloat16, 4)
    want = checkpoint_activation(x).restore()
    with launch.deferred():
        mxfp8_quantize(x)
        got = checkpoint_activation(x).restore()
        assert torch.equal(got, want)


def test_refusals():
    x = _x((4, 48), torch.bfloat16)
    with pytest.raises(ValueError, match="groups of 32"):
        checkpoint_activation(x)
    with pytest.raises(ValueError, match="at least one dimension"):
        checkpoint_activation(torch.zeros((), device=DEV))
    kept = checkpoint_activation(_x((4, 64), torch.bfloat16))
    with pytest.raises(ValueError, match="not those of codes"):
        mxfp8_dequantize(kept.codes, kept.scales[:2])
    with pytest.raises(ValueError, match="uint8 scales"):
        mxfp8_dequantize(kept.codes, kept.scales.float())
    with pytest.raises(ValueError, match="returned as"):
        kept.restore(torch.float64)
    assert "ActCheckpoint" in repr(ActCheckpoint(kept.codes, kept.scales, torch.float32))


def test_captured_and_replayed():
    x = _x((300, 256), torch.bfloat16, 5)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        checkpoint_activation(x).restore()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = checkpoint_activation(x).restore()
    for seed in range(3):
        x.copy_(_x((300, 256), torch.bfloat16, 10 + seed))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, checkpoint_activation(x).restore())
    within(out, f64(x), 2.0**-4 * f64(x).abs() + 2.0**-17 * f64(x).abs().amax(1, keepdim=True))
