"""head_norm_rope against the formula in 64 bits: both pairings, parts of a head, shared heads, positions, strides, gradients."""

from __future__ import annotations

import pytest
import torch

from oracle import cached_attention as oracle
from taac_2026_amd.api import flash_attention, head_norm_rope, rotary_table

pytestmark = pytest.mark.gpu

F32 = 2.0**-24


def _half(dtype):
    """Half a step, relative; and of the smallest numbers, absolute."""
    info = torch.finfo(dtype)
    return info.eps / 2, info.tiny * info.eps


def _inputs(device, batch, tokens, heads, kv_heads, width, dtype, seed=0, norm=True):
    g = torch.Generator().manual_seed(seed)
    q, k = (torch.randn(batch, tokens, h, width, generator=g).to(dtype).to(device).transpose(1, 2) for h in (heads, kv_heads))
    weights = [(1.0 + 0.3 * torch.randn(width, generator=g)).to(dtype).to(device) if norm else None for _ in range(2)]
    return q, k, weights


def _check_forward(got, x, weight, angles, interleaved, eps=1e-6):
    """One rounding; in float32 the statistic adds d squares (relative (d / 2 + 4) steps in the factor), a factor, a weight and the table round once each and a
    turned feature is a sum of two products: d + 16 steps of |a c| + |b s|."""
    want = oracle.head_norm_rope(x, weight, angles, eps=eps, interleaved=interleaved)
    size = oracle.head_norm_rope(x, weight, angles, eps=eps, interleaved=interleaved, magnitude=True)
    half, least = _half(got.dtype)
    bound = half * want.abs() + (x.shape[-1] + 16) * F32 * size * (1 + half) + least
    assert ((got.double() - want).abs() <= bound).all(), ((got.double() - want).abs() / bound).max()


# widths in runs of four features and others; whole heads, parts, and no rotation or norm
SHAPES = [
    (3, 17, 8, 8, 32, 32), (2, 65, 4, 2, 64, 64), (1, 1, 8, 1, 128, 64), (2, 9, 6, 3, 96, 96), (5, 3, 2, 2, 256, 128), (1, 33, 3, 1, 512, 512),
    (2, 7, 3, 3, 38, 18), (3, 5, 2, 1, 33, 32), (1, 4, 1, 1, 2, 2), (2, 6, 5, 5, 40, 20), (1, 3, 2, 2, 511, 2), (4, 2, 1, 1, 24, 8),
]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_forward(device, shape, dtype, interleaved):
    batch, tokens, heads, kv_heads, width, rotary = shape
    q, k, weights = _inputs(device, *shape[:5], dtype)
    table = rotary_table(tokens, rotary, device=device)
    angles = oracle.rotation_angles(torch.arange(tokens, device=device)[None], rotary)
    for w in (weights, [None, None]):
        got = head_norm_rope(q, k, *w, table=table, interleaved=interleaved)
        for x, out, weight in zip((q, k), got, w):
            assert out.shape == x.shape and out.transpose(1, 2).is_contiguous()
            _check_forward(out, x, weight, angles, interleaved)
    for x, out, weight in zip((q, k), head_norm_rope(q, k, *weights, eps=1e-3), weights):
        _check_forward(out, x, weight, None, interleaved, eps=1e-3)


@pytest.mark.parametrize("ints", [torch.int32, torch.int64])
def test_positions(device, ints):
    """Starts of samples, positions of tokens, far ones among them; places that the table does not have become NaN, alone."""
    q, k, weights = _inputs(device, 3, 5, 2, 1, 64, torch.float32)
    table = rotary_table(1 << 20, 32, device=device)
    starts = torch.tensor([0, 70001, (1 << 20) - 5], device=device, dtype=ints)
    positions = starts[:, None] + torch.arange(5, device=device, dtype=ints)
    for got in (head_norm_rope(q, k, *weights, table=table, starts=starts), head_norm_rope(q, k, *weights, table=table, positions=positions)):
        for x, out, weight in zip((q, k), got, weights):
            _check_forward(out, x, weight, oracle.rotation_angles(positions, 32), False)
    shared = torch.tensor([9, 3, 3, 0, 100], device=device, dtype=ints)
    for x, out, weight in zip((q, k), head_norm_rope(q, k, *weights, table=table, positions=shared), weights):
        _check_forward(out, x, weight, oracle.rotation_angles(shared[None], 32), False)
    outside = torch.tensor([-1, 1 << 20, 0], device=device, dtype=ints)
    out, _ = head_norm_rope(q, k, *weights, table=table, starts=outside)
    lost = torch.tensor([[True, False, False, False, False], [True] * 5, [False] * 5], device=device)
    assert (out[..., :32].isnan() == lost[:, None, :, None]).all() and out[..., 32:].isfinite().all()


def test_table_for_longer_contexts(device):
    """Frequencies in parts: the fast ones stay, the slow ones are divided, the table is rounded once."""
    plain = rotary_table(4096, 64, device=device).double()
    assert torch.equal(plain.float(), rotary_table(4096, 64).to(device)) or (plain - rotary_table(4096, 64).to(device).double()).abs().max() <= 2 * F32
    place = torch.arange(4096, device=device, dtype=torch.float64)[:, None]
    frequency = 10000.0 ** (-torch.arange(0, 64, 2, device=device, dtype=torch.float64) / 64)
    assert (plain[..., 0] - (place * frequency).cos()).abs().max() <= F32 and (plain[..., 1] - (place * frequency).sin()).abs().max() <= F32
    quarter = rotary_table(4096, 64, factor=4.0, device=device).double()
    assert (quarter[..., 0] - (place * frequency / 4).cos()).abs().max() <= F32
    parts = rotary_table(4096, 64, factor=4.0, trained_places=1024, magnitude=1.25, device=device).double()
    turns = 1024 * frequency / (2 * torch.pi)
    kept = ((turns - 1) / 31).clamp(0, 1)
    assert kept.max() == 1 and kept.min() == 0
    angles = place * frequency * (kept + (1 - kept) / 4)
    assert (parts[..., 1] - 1.25 * angles.sin()).abs().max() <= 2 * F32


def test_strides_and_alignment(device):
    """A packed projection's parts, rows at odd addresses, features apart, heads broadcast, the same results; the inputs stay."""
    g = torch.Generator().manual_seed(3)
    packed = torch.randn(2, 11, 3 * 4 * 32 + 8, generator=g).bfloat16().to(device)
    q, k = (packed[..., at:at + 128].unflatten(-1, (4, 32)).transpose(1, 2) for at in (0, 128))
    weight = torch.ones(32, device=device, dtype=torch.bfloat16)
    table = rotary_table(11, 32, device=device)
    want = head_norm_rope(q.contiguous(), k.contiguous(), weight, weight, table=table)
    before = packed.clone()
    odd = torch.empty(packed.numel() + 1, device=device, dtype=torch.bfloat16)[1:].view_as(packed)
    odd.copy_(packed)
    odd_q, odd_k = (odd[..., at:at + 128].unflatten(-1, (4, 32)).transpose(1, 2) for at in (0, 128))
    apart = packed.repeat_interleave(2, -1)[..., ::2]
    apart_q, apart_k = (apart[..., at:at + 128].unflatten(-1, (4, 32)).transpose(1, 2) for at in (0, 128))
    for a, b in ((q, k), (odd_q, odd_k), (apart_q, apart_k)):
        got = head_norm_rope(a, b, weight, weight, table=table)
        # the general route adds the squares in another order
        assert all((x.float() - y.float()).abs().max() <= 2.0**-7 * y.float().abs().max() for x, y in zip(got, want))
    assert torch.equal(packed, before)
    one = q[:, :1].expand(2, 4, 11, 32)
    assert torch.equal(head_norm_rope(one, one, weight, weight, table=table)[0], want[0][:, :1].expand(2, 4, 11, 32))
    # samples without tokens, no samples
    empty = head_norm_rope(q[:, :, :0], k[:, :, :0], weight, weight, table=table)
    assert empty[0].shape == (2, 4, 0, 32) and head_norm_rope(q[:0], k[:0], weight, weight, table=table)[1].shape == (0, 4, 11, 32)


def test_rows_of_zeros_and_extremes(device):
    q, k, weights = _inputs(device, 1, 4, 1, 1, 32, torch.bfloat16)
    q[:, :, 1] = 0
    q[:, :, 2] = 1e18
    q[:, :, 3, 5] = float("nan")
    out, _ = head_norm_rope(q, k, *weights, table=rotary_table(4, 32, device=device))
    assert (out[:, :, 1] == 0).all() and out[:, :, :3].isfinite().all() and out[:, :, 3].isnan().all()


def _gradients(x, weight, angles, interleaved, grad, eps=1e-6):
    """The formula's gradients in 64 bits, by autograd, and bounds. dx = rstd (w h - u mean(w h u)) with h the gradient turned back: as the forward's steps, twice, of the
    sum of sizes. dw adds `rows` products whose rounding is at most rows + d + 32 steps of the sum of their sizes."""
    leaf = x.double().requires_grad_(True)
    w = None if weight is None else weight.double().requires_grad_(True)
    out = oracle.head_norm_rope(leaf, w, angles, eps=eps, interleaved=interleaved)
    grads = torch.autograd.grad(out, [leaf] + ([] if w is None else [w]), grad.double())
    size = oracle.head_norm_rope(grad, None, None if angles is None else -angles, interleaved=interleaved, magnitude=True)
    width, rows = x.shape[-1], x[..., 0].numel()
    if weight is None:
        return grads, [4 * F32 * size]
    rstd = 1.0 / (x.double().square().mean(-1, keepdim=True) + eps).sqrt()
    unit = x.double().abs() * rstd
    part = size * weight.double().abs()
    return grads, [(2 * width + 32) * F32 * rstd * (part + unit * (part * unit).mean(-1, keepdim=True)), (rows + width + 32) * F32 * (size * unit).sum((0, 1, 2))]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [True, False])
def test_gradients(device, shape, dtype, interleaved, norm):
    batch, tokens, heads, kv_heads, width, rotary = shape
    q, k, weights = _inputs(device, *shape[:5], dtype, seed=1, norm=norm)
    grads = [torch.randn(t.shape, generator=torch.Generator().manual_seed(2)).to(dtype).to(device) for t in (q, k)]
    table = rotary_table(tokens + 50, rotary, device=device)
    starts = torch.arange(batch, device=device) * 7
    angles = oracle.rotation_angles(starts[:, None] + torch.arange(tokens, device=device), rotary)
    leaves = [t.requires_grad_(True) for t in (q, k, *weights) if t is not None]
    out = head_norm_rope(q, k, *weights, table=table, starts=starts, interleaved=interleaved)
    got = torch.autograd.grad(out, leaves, grads)
    half, least = _half(dtype)
    for i, x in enumerate((q.detach(), k.detach())):
        want, bounds = _gradients(x, weights[i] if norm else None, angles, interleaved, grads[i])
        mine = [got[i]] + ([got[2 + i]] if norm else [])
        for name, a, b, bound in zip(("x", "weight"), mine, want, bounds):
            bound = half * b.abs() + bound * (1 + half) + least
            assert ((a.double() - b).abs() <= bound).all(), (name, ((a.double() - b).abs() / bound).max())


def test_gradient_against_differences(device):
    """float64 differences of the formula along a direction, at a step where they have four digits."""
    q, k, weights = _inputs(device, 2, 3, 2, 1, 32, torch.float32, seed=4)
    grads = [torch.randn_like(t) for t in (q, k)]
    table = rotary_table(3, 32, device=device)
    angles = oracle.rotation_angles(torch.arange(3, device=device)[None], 32)
    leaves = [q, k, *weights]
    for t in leaves:
        t.requires_grad_(True)
    got = torch.autograd.grad(head_norm_rope(q, k, *weights, table=table), leaves, grads)

    def loss(q, k, wq, wk):
        return sum((oracle.head_norm_rope(x, w, angles) * g.double()).sum() for x, w, g in zip((q, k), (wq, wk), grads))

    with torch.no_grad():
        for i in range(4):
            step = torch.randn_like(leaves[i], dtype=torch.float64)
            high, low = ([t.double() + (sign * 1e-4 * step if j == i else 0.0) for j, t in enumerate(leaves)] for sign in (1, -1))
            difference = (loss(*high) - loss(*low)) / 2e-4
            # the differences' own error is 1e-8 of third derivatives of order one, rounding 1e-12; the gradient's 2^-18 of its size
            assert abs((got[i].double() * step).sum() - difference) <= 1e-4 * (got[i].double() * step).norm()


def test_one_output_alone_and_repeated(device):
    """Only one output in the loss: the other has no part; calls give the same bits."""
    q, k, weights = _inputs(device, 64, 70, 4, 2, 64, torch.bfloat16, seed=5)
    table = rotary_table(70, 64, device=device)
    leaves = [t.requires_grad_(True) for t in (q, k, *weights)]
    grad = torch.randn_like(q)
    results = []
    for _ in range(2):
        out, _ = head_norm_rope(q, k, *weights, table=table)
        results.append(torch.autograd.grad(out, leaves, grad))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert (results[0][1] == 0).all() and (results[0][3] == 0).all()
    want, bounds = _gradients(q.detach(), weights[0], oracle.rotation_angles(torch.arange(70, device=device)[None], 64), False, grad)
    assert ((results[0][2].double() - want[1]).abs() <= 2.0**-8 * want[1].abs() + 2 * bounds[1]).all()


def test_empty_backward(device):
    q, k, weights = _inputs(device, 2, 0, 2, 1, 32, torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in (q, k, *weights)]
    out = head_norm_rope(q, k, *weights, table=rotary_table(3, 32, device=device))
    got = torch.autograd.grad(out, leaves, [torch.zeros_like(t) for t in out])
    assert got[0].shape == q.shape and (got[2] == 0).all() and (got[3] == 0).all()


def test_many_rows(device):
    """More rows than workgroups: every row is reached, the weights' gradients add all of them."""
    q, k, weights = _inputs(device, 40, 1030, 8, 8, 32, torch.float32, seed=6)
    table = rotary_table(1030, 32, device=device)
    angles = oracle.rotation_angles(torch.arange(1030, device=device)[None], 32)
    leaves = [t.requires_grad_(True) for t in (q, k, *weights)]
    out = head_norm_rope(q, k, *weights, table=table, interleaved=True)
    for x, o, w in zip((q, k), out, weights):
        _check_forward(o.detach(), x.detach(), w.detach(), angles, True)
    grads = [torch.randn_like(t) for t in out]
    got = torch.autograd.grad(out, leaves, grads)
    for i, x in enumerate((q.detach(), k.detach())):
        want, bounds = _gradients(x, weights[i], angles, True, grads[i])
        for a, b, bound in zip((got[i], got[2 + i]), want, bounds):
            assert ((a.double() - b).abs() <= F32 * b.abs() + bound).all()


def test_as_many_tokens_as_there_are(device):
    """2^31 - 1 tokens, one row in memory, of which a wavefront walks sixteen thousand."""
    tokens = 2**31 - 1
    q, k = (torch.full((1, 1, 1, 1), x, device=device, dtype=torch.bfloat16).expand(1, 1, tokens, 1) for x in (2.0, -3.0))
    weights = [torch.full((1,), x, device=device, dtype=torch.bfloat16) for x in (1.5, 2.5)]
    for out, want in zip(head_norm_rope(q, k, *weights, eps=0.0), (1.5, -2.5)):
        assert out.shape == q.shape and out.min().item() == out.max().item() == want


def test_captured_with_attention(device):
    """Norm, rotation and attention, forward and backward, in a replayed graph, eager work between the replays."""
    q, k, weights = _inputs(device, 2, 40, 4, 4, 32, torch.bfloat16, seed=7)
    v = torch.randn_like(k)
    table = rotary_table(100, 32, device=device)
    starts = torch.tensor([0, 60], device=device, dtype=torch.int32)
    grad = torch.randn_like(q)
    leaves = [t.requires_grad_(True) for t in (q, k, *weights)]

    def step():
        out = flash_attention(*head_norm_rope(q, k, *weights, table=table, starts=starts), v, is_causal=True)
        return (out, *torch.autograd.grad(out, leaves, grad))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(3):
        with torch.no_grad():
            q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(seed)))
            starts.copy_(torch.tensor([seed, 3 * seed]))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, step()))


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("width,rotary", [(32, 16), (38, 18)])
def test_a_table_without_places(device, norm, width, rotary):
    """Every position lies outside: the rotated features and their gradients are NaN, the others as ever."""
    q, k, weights = _inputs(device, 2, 5, 2, 1, width, torch.float32, seed=8, norm=norm)
    leaves = [t.requires_grad_(True) for t in (q, k)]
    out = head_norm_rope(q, k, *weights, table=rotary_table(0, rotary, device=device))
    for x, o, w in zip((q, k), out, weights):
        assert o[..., :rotary].isnan().all()
        want = oracle.head_norm_rope(x.detach(), w, None)[..., rotary:]
        assert ((o[..., rotary:].double() - want).abs() <= (width + 16) * F32 * want.abs()).all()
    grads = [torch.randn_like(t) for t in out]
    for got, grad in zip(torch.autograd.grad(out, leaves, grads), grads):
        if norm:  # the mean over the head brings them all together
            assert got.isnan().all()
        else:
            assert got[..., :rotary].isnan().all() and torch.equal(got[..., rotary:], grad[..., rotary:])
