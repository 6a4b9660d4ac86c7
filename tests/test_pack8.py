"""8-bit activation checkpoints (pack8 / unpack8): bit for bit against the definition in numpy, over
types, row lengths that end inside a block, unaligned and strided inputs, blocks with infinities,
NaN or nothing but tiny values, and arrays past 2^31 values; plus the refusals."""

import numpy as np
import pytest
import torch

import spectral
from spectral import native

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def definition(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """codes and scales of float32 rows (rows, width), every operation in float32."""
    rows, width = x.shape
    blocks = -(-width // 64)
    v = np.zeros((rows, blocks * 64), np.float32)
    v[:, :width] = x
    v = v.reshape(rows, blocks, 64)
    with np.errstate(all="ignore"):
        m = np.maximum(np.abs(v).max(-1, keepdims=True), np.float32(2.0 ** -100))
        codes = np.rint(v * (np.float32(127.0) / m))
        scales = (m / np.float32(127.0))[..., 0]
    bad = ~np.isfinite(v).all(-1)
    codes[bad] = 0
    scales[bad] = np.nan
    return codes.reshape(rows, -1)[:, :width].astype(np.int8), scales


def values(rows, width, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, width, generator=g) * torch.exp(2.0 * torch.randn(rows, 1, generator=g))
    return x.to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("rows", "width"), [(1, 1), (3, 7), (5, 63), (4, 64), (7, 65), (1000, 130), (33, 72),
                                             (257, 128), (2, 4099)])
def test_codes_scales_and_values_are_the_definition_s(rows, width, dtype):
    x = values(rows, width, dtype, rows * 131 + width)
    codes, scales = spectral.pack8(x.cuda())
    want_codes, want_scales = definition(x.float().numpy())
    assert codes.dtype == torch.int8 and scales.shape == (rows, -(-width // 64))
    np.testing.assert_array_equal(codes.cpu().numpy(), want_codes)
    np.testing.assert_array_equal(scales.cpu().numpy(), want_scales)
    step = np.repeat(want_scales, 64, axis=1)[:, :width]
    for out in DTYPES:
        back = spectral.unpack8(codes, scales, dtype=out).cpu()
        assert torch.equal(back, torch.from_numpy(want_codes.astype(np.float32) * step).to(out))
    # Half a step, and the roundings of the product and of code * scale (2^-22 of the block's largest).
    err = np.abs(spectral.unpack8(codes, scales).cpu().numpy().astype(np.float64) - x.double().numpy())
    assert (err <= step.astype(np.float64) * (0.5 + 127 * 2.0 ** -22)).all()


@pytest.mark.gpu
def test_blocks_that_hold_no_ordinary_number():
    x = torch.zeros(6, 130)
    x[1, 70] = float("inf")
    x[2, 3] = float("nan")
    x[3, :64] = 1e-40           # below the smallest scale
    x[4, 129] = torch.finfo(torch.float32).max
    x[5, 0] = -float("inf")
    x[:, 5] += 0.5
    codes, scales = spectral.pack8(x.cuda())
    want_codes, want_scales = definition(x.numpy())
    np.testing.assert_array_equal(codes.cpu().numpy(), want_codes)
    np.testing.assert_array_equal(scales.cpu().numpy(), want_scales)
    back = spectral.unpack8(codes, scales).cpu()
    assert back[1, 64:128].isnan().all() and back[1, :64].isfinite().all()
    assert back[2, :64].isnan().all() and back[5, :64].isnan().all()
    assert back[4].isfinite().all()


@pytest.mark.gpu
def test_views_and_empty_arrays():
    base = values(40, 200, torch.bfloat16, 5).cuda()
    for x in (base[:, 3:131], base.t(), base[1::2], base.view(-1)[1:1 + 64 * 8].view(8, 64)):
        codes, scales = spectral.pack8(x)
        want = spectral.pack8(x.contiguous().clone())
        assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])
        assert torch.equal(spectral.unpack8(codes.t().contiguous().t(), scales), spectral.unpack8(*want))
    for shape in [(0, 64), (4, 0), (0,)]:
        codes, scales = spectral.pack8(torch.zeros(shape, device="cuda"))
        assert codes.shape == shape and spectral.unpack8(codes, scales).shape == shape


@pytest.mark.gpu
def test_on_a_side_stream():
    x = values(4096, 256, torch.float32, 9).cuda()
    want = spectral.pack8(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        codes, scales = spectral.pack8(x * 1.0)
    side.synchronize()
    assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])


@pytest.mark.gpu
def test_past_two_to_the_31_values():
    rows = (1 << 25) + 3
    x = torch.zeros(rows, 64, dtype=torch.bfloat16, device="cuda")
    tail = values(5, 64, torch.bfloat16, 1)
    x[-5:] = tail.cuda()
    codes, scales = spectral.pack8(x)
    want_codes, want_scales = definition(tail.float().numpy())
    np.testing.assert_array_equal(codes[-5:].cpu().numpy(), want_codes)
    np.testing.assert_array_equal(scales[-5:].cpu().numpy(), want_scales)
    del x
    back = spectral.unpack8(codes, scales, dtype=torch.bfloat16)
    assert torch.equal(back[-5:].cpu(), torch.from_numpy(want_codes.astype(np.float32) * want_scales).to(torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("width", [2 ** 31 - 8, 2 ** 31 - 1])  # whole 16-byte pieces, and not
def test_the_longest_rows(width):
    first = (width - 1) // 64 * 64 - 128  # of the last blocks
    tail = values(1, width - first, torch.float16, 3)
    x = torch.zeros(1, width, dtype=torch.float16, device="cuda")
    x[0, first:] = tail[0].cuda()
    codes, scales = spectral.pack8(x)
    want_codes, want_scales = definition(tail.float().numpy())
    np.testing.assert_array_equal(codes[:, first:].cpu().numpy(), want_codes)
    np.testing.assert_array_equal(scales[:, first // 64:].cpu().numpy(), want_scales)
    assert not codes[:, :first].any()
    del x
    back = spectral.unpack8(codes, scales, dtype=torch.float16)
    step = np.repeat(want_scales, 64, axis=1)[:, :width - first]
    assert torch.equal(back[:, first:].cpu(), torch.from_numpy(want_codes.astype(np.float32) * step).to(torch.float16))


@pytest.mark.parametrize(
    ("fn", "args", "message"),
    [
        ("spectral_pack8", (4096, 3, 8192, 16384, 1, 64, None), "dtype must be"),
        ("spectral_pack8", (4096, 0, 8192, 16384, -1, 64, None), "rows >= 0"),
        ("spectral_pack8", (4096, 0, None, 16384, 1, 64, None), "null array"),
        ("spectral_pack8", (4097, 1, 8192, 16384, 1, 64, None), "aligned"),
        ("spectral_unpack8", (4096, 8194, 8192, 0, 1, 64, None), "aligned"),
        ("spectral_unpack8", (4096, 8192, 8192, 7, 1, 64, None), "dtype must be"),
    ],
)
def test_the_c_abi_refuses(fn, args, message):
    with pytest.raises(ValueError, match=message):
        native.call(fn, *args)


def test_cpu_tensors_are_refused():
    with pytest.raises(NotImplementedError, match="CPU"):
        spectral.pack8(torch.zeros(2, 64))


@pytest.mark.gpu
def test_wrong_types_and_shapes_are_refused():
    x = torch.zeros(2, 70, device="cuda")
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        spectral.pack8(x.double())
    with pytest.raises(RuntimeError, match="at least one dimension"):
        spectral.pack8(x[0, 0])
    codes, scales = spectral.pack8(x)
    with pytest.raises(RuntimeError, match="scales must be float32 of shape"):
        spectral.unpack8(codes, scales[:, :1])
    with pytest.raises(RuntimeError, match="codes must be an int8"):
        spectral.unpack8(x, scales)
    with pytest.raises(RuntimeError, match="the result must be"):
        spectral.unpack8(codes, scales, dtype=torch.float64)
