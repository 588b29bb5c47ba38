"""Rotary positions on the GPU against the oracle in 64 bits.

Error: cosine and sine are rounded to fp32 (2^-24 relative each), and so are the two products and their sum (one rounding
fewer where they are fused): within 4 * 2^-24 of |x c| + |y s|; then half a step of the rows' type (fp16 below 2^-14: half of 2^-24)."""

import numpy as np
import pytest
import torch

from conftest import announce
from oracle import rotary as ora

pytestmark = pytest.mark.gpu

STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 0.0}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0**-25, torch.float32: 2.0**-140}


def _near(got, x, positions, frequencies, interleaved, factor):
    x = x.double().cpu().numpy()
    want = ora.rotated(x, positions.cpu().numpy(), frequencies.cpu().numpy(), interleaved, factor)
    half = len(frequencies)
    size = np.zeros_like(x)  # |x c| + |y s| is at most factor sqrt(x^2 + y^2) sqrt 2
    one, two = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    size[..., one] = size[..., two] = abs(factor) * np.sqrt(2 * (x[..., one] ** 2 + x[..., two] ** 2))
    mid = 4 * 2.0**-24 * size
    bound = mid + STEP[got.dtype] * (np.abs(want) + mid) + TINY[got.dtype]
    far = np.abs(got.double().cpu().numpy() - want)
    assert (far <= bound).all(), float((far - bound).max())
    assert np.array_equal(got.double().cpu().numpy()[..., 2 * half:], x[..., 2 * half:])


def _run(dev, tokens, hq, hk, dim, half, dtype, interleaved, far, seed=0, factor=1.0, in_place=False, index=torch.int64):
    from eagle_harness.vllm.rotary import rotate_rows, rotary_frequencies

    gen = torch.Generator().manual_seed(seed)
    q = torch.randn(tokens, hq, dim, generator=gen).to(dtype)
    k = torch.randn(tokens, hk, dim, generator=gen).to(dtype) if hk else None
    positions = torch.randint(0, far, (tokens,), generator=gen).to(index)
    frequencies, _ = rotary_frequencies(2 * half, 10000.0, device=dev)
    a, b = q.to(dev), None if k is None else k.to(dev)
    outs = {} if in_place else dict(q_out=torch.full_like(a, 9.0), k_out=None if b is None else torch.full_like(b, 9.0))
    x, y = rotate_rows(a, b, positions.to(dev), frequencies, interleaved=interleaved, factor=factor, **outs)
    torch.cuda.synchronize()
    assert x is (a if in_place else outs["q_out"])
    _near(x, q, positions, frequencies, interleaved, factor)
    if hk:
        _near(y, k, positions, frequencies, interleaved, factor)
    if not in_place:
        assert torch.equal(a.cpu(), q)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,hq,hk,dim,half", [(1, 1, 1, 2, 1), (1, 8, 2, 64, 32), (16, 24, 4, 256, 32), (3, 5, 1, 80, 20),
                                                   (7, 3, 3, 13, 5), (1030, 16, 1, 128, 64), (2, 2, 0, 576, 32), (5, 1, 1, 1100, 512),
                                                   (600, 3, 2, 96, 12)])
def test_layouts_and_sizes(dev, tokens, hq, hk, dim, half, dtype, interleaved):
    announce(f"rotary {tokens}x{hq}/{hk}x{dim} half={half} {dtype} interleaved={interleaved}")
    _run(dev, tokens, hq, hk, dim, half, dtype, interleaved, 5000, seed=tokens + dim)
    _run(dev, tokens, hq, hk, dim, half, dtype, interleaved, 5000, seed=1, in_place=True, factor=1.25, index=torch.int32)


@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions_keep_their_angle(dev, interleaved):
    announce("rotary far positions")
    _run(dev, 300, 4, 2, 128, 64, torch.float32, interleaved, 1 << 22)
    _run(dev, 300, 4, 2, 128, 64, torch.float32, interleaved, (1 << 31) - 1)


def test_positions_zero_and_below(dev):
    from eagle_harness.vllm.rotary import rotate_rows, rotary_frequencies

    announce("rotary position 0 and negative ones")
    f, _ = rotary_frequencies(64, device=dev)
    q = torch.randn(3, 2, 64, device=dev)
    x, _ = rotate_rows(q, None, torch.zeros(3, dtype=torch.int32, device=dev), f, q_out=torch.empty_like(q))
    assert torch.equal(x, q)
    positions = torch.tensor([-1, -77, -100000], device=dev)
    x, _ = rotate_rows(q, None, positions, f, q_out=torch.empty_like(q))
    _near(x, q, positions, f, False, 1.0)


@pytest.mark.parametrize("offset", [0, 1, 4])
@pytest.mark.parametrize("interleaved", [False, True])
def test_parts_of_a_packed_projection(dev, interleaved, offset):
    """q and k as views of one [tokens, q | k | v] buffer, on and off 16-byte boundaries; the rest of it stays."""
    from eagle_harness.vllm.rotary import rotate_rows, rotary_frequencies

    announce(f"rotary packed offset={offset}")
    tokens, hq, hk, dim = 37, 6, 2, 64
    width = (hq + 2 * hk) * dim + offset
    store = torch.randn(tokens, width, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    f, _ = rotary_frequencies(32, 1e6, device=dev)
    positions = torch.arange(100, 100 + tokens, device=dev)
    buf = store.to(dev)
    view = lambda t: (t[:, offset:offset + hq * dim].unflatten(1, (hq, dim)),  # noqa: E731
                      t[:, offset + hq * dim:offset + (hq + hk) * dim].unflatten(1, (hk, dim)))
    q, k = view(buf)
    rotate_rows(q, k, positions, f, interleaved=interleaved)
    want_q, want_k = view(store)
    _near(q, want_q, positions, f, interleaved, 1.0)
    _near(k, want_k, positions, f, interleaved, 1.0)
    assert torch.equal(buf[:, :offset].cpu(), store[:, :offset])
    assert torch.equal(buf[:, offset + (hq + hk) * dim:].cpu(), store[:, offset + (hq + hk) * dim:])
    # heads outside tokens, and a head that follows at another stride
    x = torch.randn(hq, tokens, dim, device=dev).transpose(0, 1)
    y, _ = rotate_rows(x, None, positions, f, interleaved=interleaved, q_out=torch.empty(tokens, hq, dim, device=dev))
    _near(y, x, positions, f, interleaved, 1.0)


def test_infinities_and_nan_stay_in_their_pair(dev):
    from eagle_harness.vllm.rotary import rotate_rows, rotary_frequencies

    announce("rotary infinities")
    f, _ = rotary_frequencies(8, device=dev)
    q = torch.ones(1, 2, 16, device=dev)
    q[0, 0, 1] = torch.nan
    q[0, 1, 15] = torch.inf
    x, _ = rotate_rows(q, None, torch.tensor([5], device=dev), f, q_out=torch.empty_like(q))
    assert torch.isnan(x[0, 0, [1, 5]]).all() and torch.isfinite(x[0, 0, [0, 2, 3, 4, 6, 7]]).all()
    assert x[0, 1, 15] == torch.inf and torch.isfinite(x[0, 1, :15]).all()


def test_scaled_frequencies_and_replayed(dev):
    from eagle_harness.vllm.rotary import rotate_rows, rotary_frequencies

    announce("rotary scaled, captured")
    q, k = torch.randn(9, 4, 128, device=dev), torch.randn(9, 2, 128, device=dev)
    a, b = torch.empty_like(q), torch.empty_like(k)
    positions = torch.arange(9, device=dev)
    f, factor = rotary_frequencies(128, scaling="yarn", stretch=8.0, trained=4096, device=dev)
    rotate_rows(q, k, positions, f, factor=factor, q_out=a, k_out=b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rotate_rows(q, k, positions, f, factor=factor, q_out=a, k_out=b)
    for i in range(3):
        positions += 1000
        q.normal_()
        graph.replay()
        _near(a, q, positions, f, False, factor)
        _near(b, k, positions, f, False, factor)


def test_no_rows_and_no_heads(dev):
    from eagle_harness.vllm.rotary import rotate_rows, rotary_frequencies

    f, _ = rotary_frequencies(8, device=dev)
    at = torch.zeros(0, dtype=torch.int64, device=dev)
    assert rotate_rows(torch.empty(0, 4, 8, device=dev), None, at, f)[0].shape == (0, 4, 8)
    q, k = torch.empty(2, 0, 8, device=dev), torch.randn(2, 3, 8, device=dev)
    want = k.clone()
    rotate_rows(q, k, torch.zeros(2, dtype=torch.int64, device=dev), f)
    assert torch.equal(k, want)
