"""Operators of the packed training step: packed attention with gradients,
cross-entropy, gradient norm and clipping. Everything is held to plain 64-bit
arithmetic, with bounds that count the roundings a result goes through.

The units: H = 2^-8, half a step of bf16 (2^-11 for fp16), and E = 2^-11 for
all fp32 arithmetic on the way to a sum (a score is a sum of at most 128
products: 128 * 2^-24 = 2^-17 of sum |q||k| scale, which is below 20 at these
inputs, so a probability is off by less than 2^-12 of itself, twice)."""
import math
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from runbookai_amd import ops
from runbookai_amd.ops import reference

H, E = 2.0 ** -8, 2.0 ** -11

gpu = pytest.mark.gpu


def _starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


# ---------------------------------------------------------- packed attention

def attention_oracle(q, k, v, dout, starts, scale):
    """(out, dq, dk, dv) in 64 bits, and how far a kernel may be off each:
    operands P and dS rounded once, the result once, delta from a rounded o
    beyond a sequence's first 128 rows."""
    q, k, v, dout = (x.detach().double().cpu() for x in (q, k, v, dout))
    group = q.shape[1] // k.shape[1]
    out, dq, dk, dv = (torch.zeros_like(x) for x in (q, q, k, v))
    tol = [torch.zeros_like(x) for x in (q, q, k, v)]
    for a, b in zip(starts[:-1], starts[1:]):
        n = b - a
        for h in range(q.shape[1]):
            g = h // group
            qs, ks, vs, do = q[a:b, h], k[a:b, g], v[a:b, g], dout[a:b, h]
            s = (qs @ ks.T) * scale
            s = s.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), -math.inf)
            p = s.softmax(-1)
            o = p @ vs
            dp = do @ vs.T
            delta = (p * dp).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            out[a:b, h] = o
            dq[a:b, h] = ds @ ks * scale
            dk[a:b, g] += ds.T @ qs * scale
            dv[a:b, g] += p.T @ do
            reach = p @ vs.abs()
            tol[0][a:b, h] = (H + E) * reach + H * (o.abs() + H * reach)
            # |error of dS| before its own rounding
            far = (torch.arange(n) >= 128).double()[:, None]
            e = E * p * (do.abs() @ vs.abs().T + delta.abs())
            e = e + p * far * 2 * H * (do.abs() * reach).sum(-1, keepdim=True)
            e = e + H * (ds.abs() + e)
            tol[1][a:b, h] = e @ ks.abs() * scale * (1 + H) + H * dq[a:b, h].abs()
            tol[2][a:b, g] += e.T @ qs.abs() * scale * (1 + H)
            tol[3][a:b, g] += (H + E) * (p.T @ do.abs()) * (1 + H)
    tol[2] += H * dk.abs()
    tol[3] += H * dv.abs()
    return (out, dq, dk, dv), tol


def _inputs(lens, heads, d, pad=0, device="cpu", dtype=torch.bfloat16, seed=0):
    gen = torch.Generator().manual_seed(seed)
    T = sum(lens) + pad
    hq, hk = heads
    mk = lambda h, std: (torch.randn(T, h, d, generator=gen) * std).to(dtype).to(device)  # noqa: E731
    return mk(hq, 1.0), mk(hk, 1.0), mk(hk, 1.0), mk(hq, 0.1)


def _attend(q, k, v, dout, starts, scale=None):
    q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
    out = ops.packed_attention(q, k, v, starts, scale=scale)
    return (out.detach(), *torch.autograd.grad(out, (q, k, v), dout))


def _within(got, want, tol, names=("out", "dq", "dk", "dv")):
    for name, x, y, t in zip(names, got, want, tol):
        x = x.double().cpu()
        assert torch.isfinite(x).all(), name
        over = (x - y).abs() - t
        assert (over <= 1e-30).all(), (name, float(over.max()), int((over > 0).sum()))


LENGTHS = [
    [1], [2], [31], [32, 33], [63, 64, 65], [127, 128, 129], [0, 1, 0, 0, 5, 0],
    [257, 3, 640], [1] * 70, [1000],
]


@pytest.mark.parametrize("lens", [[1], [5, 0, 3], [0], [7, 20]])
@pytest.mark.parametrize("heads", [(4, 2), (3, 3)])
def test_attention_reference(lens, heads):
    q, k, v, dout = _inputs(lens, heads, 8, pad=2, dtype=torch.float64)
    starts = torch.tensor(_starts(lens), dtype=torch.int32)
    want, _ = attention_oracle(q, k, v, dout, starts.tolist(), 0.4)
    for x, y in zip(_attend(q, k, v, dout, starts, 0.4), want):
        torch.testing.assert_close(x, y, rtol=1e-12, atol=1e-12)


def test_attention_reference_without_sequences():
    q, k, v, dout = _inputs([3], (2, 1), 4)
    assert not any(x.any() for x in _attend(q, k, v, dout, torch.tensor([0])))


def test_attention_reference_gradcheck():
    q, k, v, _ = _inputs([4, 3], (2, 1), 4, pad=1, dtype=torch.float64)
    starts = torch.tensor([0, 4, 7])
    assert torch.autograd.gradcheck(
        lambda *a: ops.packed_attention(*a, starts), [x.requires_grad_() for x in (q, k, v)])


def test_attention_reference_agrees_with_prefill():
    q, k, v, _ = _inputs([9, 14], (4, 2), 64)
    starts = torch.tensor([0, 9, 23], dtype=torch.int32)
    a = ops.packed_attention(q, k, v, starts)
    b = reference.prefill_attention(q, k, v, starts)
    assert torch.equal(a, b)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_attention_refuses(device):
    q, k, v, _ = _inputs([4], (4, 2), 64, device=device)
    starts = torch.tensor([0, 4], dtype=torch.int32)
    call = ops.packed_attention
    bad = [
        (q[0], k, v, starts), (q, k[:3], v, starts), (q, k, v[:, :1], starts),
        (q[:, :3], k, v, starts), (q, k.float(), v, starts), (q, k[:, :0], v[:, :0], starts),
        (q, k, v, starts.float()), (q, k, v, starts[None]), (q, k, v, starts[:0]),
        (q, k, v, torch.tensor([0, 5])), (q, k, v, torch.tensor([-1, 4])),
        (q, k, v, torch.tensor([0, 3, 2])),
    ]
    for args in bad:
        with pytest.raises(ValueError):
            call(*args)
    for scale in (0.0, -1.0, math.inf, math.nan, 1e39):
        with pytest.raises(ValueError):
            call(q, k, v, starts, scale=scale)
    with pytest.raises(ValueError):
        call(q[..., :0], k[..., :0], v[..., :0], starts)
    if device == "cuda":
        with pytest.raises(ValueError):
            call(q.float(), k.float(), v.float(), starts)
        with pytest.raises(ValueError):
            call(q[..., :32], k[..., :32], v[..., :32], starts)
        with pytest.raises(ValueError):
            call(q, k.cpu(), v, starts)


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads", [(4, 2), (3, 3), (6, 2), (8, 1)])
@pytest.mark.parametrize("lens", LENGTHS, ids=lambda x: "-".join(map(str, x))[:20])
def test_attention_gpu(lens, heads, d):
    q, k, v, dout = _inputs(lens, heads, d, pad=5, device="cuda")
    starts = _starts(lens)
    got = _attend(q, k, v, dout, torch.tensor(starts, dtype=torch.int32, device="cuda"))
    want, tol = attention_oracle(q, k, v, dout, starts, 1.0 / math.sqrt(d))
    _within(got, want, tol)
    end = starts[-1]
    assert all(not x[end:].any() for x in got)   # rows in no sequence
    with torch.no_grad():
        plain = ops.packed_attention(q, k, v, torch.tensor(starts))
    assert torch.equal(plain, got[0])


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens,heads", [
    ([257, 3, 640], (32, 8)),      # enough workgroups for one wave set a tile
    ([257, 3, 640], (64, 64)),     # and for dk, dv
    ([900, 130, 77], (64, 8)),     # more than run at once: a table of tiles
    ([9] * 100, (4, 2)),           # more sequences than a wave looks through
    ([128] * 70, (6, 3)),
])
def test_attention_gpu_large_grids(lens, heads, d):
    q, k, v, dout = _inputs(lens, heads, d, pad=5, device="cuda")
    starts = _starts(lens)
    got = _attend(q, k, v, dout, torch.tensor(starts, dtype=torch.int32, device="cuda"))
    want, tol = attention_oracle(q, k, v, dout, starts, 1.0 / math.sqrt(d))
    _within(got, want, tol)
    assert all(not x[starts[-1]:].any() for x in got)


@gpu
@pytest.mark.parametrize("lens,heads,d", [
    ([2300], (8, 1), 64), ([1, 1900, 130], (4, 4), 64), ([700] * 4, (4, 2), 64),
    ([1500, 40, 700], (8, 2), 128), ([300] * 5 + [2000], (16, 2), 128), ([1100], (2, 2), 128)])
def test_attention_gpu_split_gradients(lens, heads, d):
    """Long sequences in few tiles, whose dk and dv are summed by several
    workgroups: right, and the same bits every time."""
    q, k, v, dout = _inputs(lens, heads, d, pad=5, device="cuda")
    starts = torch.tensor(_starts(lens), dtype=torch.int32, device="cuda")
    got = _attend(q, k, v, dout, starts)
    want, tol = attention_oracle(q, k, v, dout, _starts(lens), 1.0 / math.sqrt(d))
    _within(got, want, tol)
    for _ in range(20):
        for x, y in zip(_attend(q, k, v, dout, starts), got):
            assert torch.equal(x, y)


@gpu
@pytest.mark.parametrize("lens,heads,d", [
    ([1500, 0, 700, 64, 1, 1300], (8, 4), 64), ([4000], (32, 8), 128), ([129] * 62, (16, 2), 64),
    ([129] * 63, (16, 2), 64), (list(range(20, 320, 5)), (8, 8), 128)])
def test_attention_gpu_forward_alone(lens, heads, d):
    """Without gradients to come, tiles are found another way: the same bits."""
    q, k, v, dout = _inputs(lens, heads, d, pad=200, device="cuda")
    starts = torch.tensor(_starts(lens), dtype=torch.int32, device="cuda") + 100
    want = _attend(q, k, v, dout, starts)[0]
    q[:100] = math.nan
    q[100 + sum(lens):] = math.nan
    with torch.no_grad():
        assert torch.equal(ops.packed_attention(q, k, v, starts), want)


@gpu
@pytest.mark.parametrize("d", [64, 128])
def test_attention_gpu_sharp_scores(d):
    """Scores far apart: the running maximum grows many times, and most
    probabilities underflow."""
    lens = [300, 41]
    q, k, v, dout = _inputs(lens, (4, 2), d, device="cuda")
    ramp = torch.linspace(0.1, 8.0, sum(lens), device="cuda")[:, None, None]
    k = (k * ramp).to(torch.bfloat16)
    starts = _starts(lens)
    got = _attend(q, k, v, dout, torch.tensor(starts, device="cuda"))
    want, tol = attention_oracle(q, k, v, dout, starts, 1.0 / math.sqrt(d))
    # sum |q||k| scale is 8 times what E counts with
    _within(got, want, [8 * t for t in tol])


@gpu
@pytest.mark.parametrize("d", [64, 128])
def test_attention_gpu_views(d):
    """q, k, v as slices of one projection, an expanded and a misaligned one,
    and a broadcast gradient."""
    lens, hq, hk = [70, 1, 130], 4, 2
    T, starts = sum(lens), torch.tensor(_starts(lens), dtype=torch.int32, device="cuda")
    gen = torch.Generator().manual_seed(3)
    qkv = torch.randn(T, (hq + 2 * hk) * d, generator=gen).to(torch.bfloat16).cuda()
    q, k, v = (x.view(T, -1, d) for x in qkv.split([hq * d, hk * d, hk * d], -1))
    dout = (torch.randn(T, 1, 1, generator=gen) * 0.1).to(torch.bfloat16).cuda().expand(T, hq, d)
    dense = _attend(*(x.contiguous() for x in (q, k, v, dout)), starts)
    for x, y in zip(_attend(q, k, v, dout, starts), dense):
        assert torch.equal(x, y)
    off = torch.empty(T * hk * d + 1, dtype=torch.bfloat16, device="cuda")[1:].view(T, hk, d)
    off.copy_(k)
    turned = v.transpose(0, 1).contiguous().transpose(0, 1)
    for x, y in zip(_attend(q, off, turned, dout, starts), dense):
        assert torch.equal(x, y)
    one = k[:, :1].expand(T, hk, d)
    got = _attend(q, one, v, dout, starts)
    for x, y in zip(got, _attend(q, one.contiguous(), v, dout, starts)):
        assert torch.equal(x, y)


@gpu
def test_attention_gpu_fused_projection_gradient():
    """The gradient arrives in the tensor that q, k and v are slices of."""
    T, hq, hk, d = 90, 4, 2, 64
    starts = torch.tensor([0, 40, 90], device="cuda")
    x = torch.randn(T, (hq + 2 * hk) * d, device="cuda").to(torch.bfloat16).requires_grad_()
    parts = [p.view(T, -1, d) for p in x.split([hq * d, hk * d, hk * d], -1)]
    out = ops.packed_attention(*parts, starts)
    dout = torch.randn_like(out)
    out.backward(dout)
    got = _attend(*(p.detach() for p in parts), dout, starts)[1:]
    assert torch.equal(x.grad, torch.cat([g.reshape(T, -1) for g in got], -1))


@gpu
def test_attention_gpu_not_finite_elsewhere():
    """What other sequences and unused rows hold changes nothing."""
    lens, d = [60, 200, 1], 64
    starts = torch.tensor([10, 70, 270, 271], dtype=torch.int32, device="cuda")
    q, k, v, dout = _inputs(lens, (4, 2), d, pad=29, device="cuda")
    clean = _attend(q, k, v, dout, starts)
    for x in (q, k, v, dout):
        x[:10] = math.nan
        x[70:270, :, ::3] = math.inf
        x[271:] = math.nan
    got = _attend(q, k, v, dout, starts)
    for x, y in zip(got, clean):
        assert torch.equal(x[10:70], y[10:70]) and torch.equal(x[270], y[270])
        assert not x[:10].any() and not x[271:].any()


@gpu
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("heads", [(4, 2), (128, 2)])   # without and with a table of tiles
@pytest.mark.parametrize("starts", [[0, 300], [0, 120, 60, 200], [-4, 200], [5, 3],
                                    [0, 2 ** 32 + 200], [0] + [150, 100] * 40])
def test_attention_gpu_wrong_starts(starts, heads, dtype):
    if dtype == torch.int32 and max(starts) > 2 ** 31:
        pytest.skip("no 32-bit value")
    q, k, v, dout = _inputs([200], heads, 64, device="cuda")
    got = _attend(q, k, v, dout, torch.tensor(starts, dtype=dtype, device="cuda"))
    assert all(torch.isnan(x).all() for x in got)


@gpu
@pytest.mark.parametrize("heads", [(4, 2), (128, 2)])
def test_attention_gpu_starts_may_change_before_the_backward_pass(heads):
    """A buffer of starts that the next batch is written to."""
    q, k, v, dout = _inputs([100, 60], heads, 64, device="cuda")
    starts = torch.tensor([0, 100, 160], dtype=torch.int32, device="cuda")
    want = _attend(q, k, v, dout, starts.clone())
    parts = [x.detach().requires_grad_() for x in (q, k, v)]
    out = ops.packed_attention(*parts, starts)
    starts.copy_(torch.tensor([0, 7, 8], dtype=torch.int32))
    got = torch.autograd.grad(out, parts, dout)
    assert all(torch.equal(x, y) for x, y in zip(got, want[1:]))


@gpu
def test_attention_gpu_two_passes_over_one_graph():
    q, k, v, dout = _inputs([100, 60], (4, 2), 64, device="cuda")
    starts = torch.tensor([0, 100, 160], device="cuda")
    parts = [x.detach().requires_grad_() for x in (q, k, v)]
    out = ops.packed_attention(*parts, starts)
    other = torch.randn_like(dout)
    a = torch.autograd.grad(out, parts, dout, retain_graph=True)
    b = torch.autograd.grad(out, parts, other, retain_graph=True)
    c = torch.autograd.grad(out, parts, dout)
    assert all(torch.equal(x, y) for x, y in zip(a, c))
    want = _attend(q, k, v, other, starts)[1:]
    assert all(torch.equal(x, y) for x, y in zip(b, want))


@gpu
def test_attention_gpu_nothing():
    q, k, v, dout = _inputs([0], (4, 2), 64, device="cuda")
    for starts in ([0], [0, 0, 0]):
        got = _attend(q, k, v, dout, torch.tensor(starts, device="cuda"))
        assert [x.shape[0] for x in got] == [0] * 4
    q, k, v, dout = _inputs([3], (4, 2), 64, device="cuda")
    assert not any(x.any() for x in _attend(q, k, v, dout, torch.tensor([0], device="cuda")))


@gpu
def test_attention_gpu_repeats_bit_for_bit_on_another_stream():
    q, k, v, dout = _inputs([500, 77, 300], (8, 2), 128, device="cuda")
    starts = torch.tensor([0, 500, 577, 877], device="cuda")
    want = _attend(q, k, v, dout, starts)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = _attend(q, k, v, dout, starts)
    b = _attend(k.repeat_interleave(4, 1), k, v, dout, starts)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(a, want))
    assert not torch.equal(b[0], want[0])


@gpu
@pytest.mark.parametrize("T,cuts", [
    (400, ([100, 100, 380], [1, 399, 400], [0, 0, 256])),
    (2100, ([2100] * 3, [1, 1000, 1100], [0, 0, 1700], [600, 1200, 2100], [2100] * 3))])
def test_attention_gpu_captured(T, cuts):
    """Forward and backward in one graph: new data and new sequences in the
    same buffers, replayed between eager calls."""
    q, k, v, dout = _inputs([T], (4, 2), 64, device="cuda")
    starts = torch.tensor([0, 100, 100, 380], dtype=torch.int32, device="cuda")
    leaves = [x.requires_grad_() for x in (q, k, v)]

    def step():
        out = ops.packed_attention(*leaves, starts)
        return (out, *torch.autograd.grad(out, leaves, dout))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for i, ends in enumerate(cuts):
        with torch.no_grad():
            for x, y in zip((q, k, v, dout), _inputs([T], (4, 2), 64, device="cuda", seed=i)):
                x.copy_(y)
            starts.copy_(torch.tensor([0] + ends, dtype=torch.int32))
        graph.replay()
        got = [x.detach().clone() for x in static]
        for x, y in zip(got, _attend(q, k, v, dout, starts)):
            assert torch.equal(x, y)
        torch.cuda.synchronize()


@gpu
def test_attention_gpu_gradient_against_differences():
    """The gradients against differences of the loss in 64 bits."""
    lens, d = [50, 150], 64
    q, k, v, dout = _inputs(lens, (4, 2), d, device="cuda")
    starts = _starts(lens)
    got = _attend(q, k, v, dout, torch.tensor(starts, device="cuda"))[1:]
    base = [x.double().cpu() for x in (q, k, v)]
    gen = torch.Generator().manual_seed(1)

    def loss(parts):
        out = reference.packed_attention(*parts, torch.tensor(starts), 1 / math.sqrt(d))
        return float((out * dout.double().cpu()).sum())

    _, tol = attention_oracle(q, k, v, dout, starts, 1 / math.sqrt(d))
    for i in range(3):
        way = torch.randn(base[i].shape, generator=gen, dtype=torch.float64)
        h = 1e-5
        up, down = ([b + s * h * way if j == i else b for j, b in enumerate(base)]
                    for s in (1, -1))
        slope = (loss(up) - loss(down)) / (2 * h)
        mine = float((got[i].double().cpu() * way).sum())
        # what the bound allows each element, and 1e-6 for the third derivative
        assert abs(mine - slope) <= float((tol[i + 1] * way.abs()).sum()) + 1e-6


@gpu
def test_attention_gpu_long():
    """One sequence of many tiles; rows far apart in the result are checked."""
    T, d = 20000, 64
    q, k, v, _ = _inputs([T], (2, 1), d, device="cuda")
    with torch.no_grad():
        out = ops.packed_attention(q, k, v, torch.tensor([0, T], device="cuda"))
    for row in (0, 127, 128, 9999, 16383, T - 1):
        ks, vs = k[:row + 1, 0].double(), v[:row + 1, 0].double()
        p = (q[row].double() @ ks.T / math.sqrt(d)).softmax(-1)
        want, reach = p @ vs, p @ vs.abs()
        assert ((out[row].double() - want).abs() <= (H + E) * reach + H * want.abs() + H * H).all()


# ------------------------------------------------------------- cross-entropy

def loss_oracle(x, targets, reduction, gout, ignore=-100):
    x = x.detach().double().cpu().requires_grad_()
    t = targets.cpu()
    real = t != ignore
    each = torch.zeros(t.shape, dtype=torch.float64)
    each[real] = (x.logsumexp(-1) - x.gather(1, t.clamp(min=0).long()[:, None])[:, 0])[real]
    loss = {"none": each, "sum": each.sum(), "mean": each.sum() / real.sum()}[reduction]
    grad, = torch.autograd.grad(loss, x, gout.double().cpu())
    return loss.detach(), grad


SIZES = [(1, 1), (3, 2), (5, 7), (4, 64), (9, 511), (2, 4096), (3, 4099), (5, 8192), (2, 8193),
         (2, 20001), (1, 128256)]
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _loss_inputs(n, v, dtype, device, seed=0, labelled=0.6):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, v, generator=gen) * 3).to(dtype).to(device)
    t = torch.randint(0, v, (n,), generator=gen)
    t[torch.rand(n, generator=gen) >= labelled] = -100
    t[0] = v - 1
    return x, t.to(device)


def _loss_and_grad(x, t, reduction, gout=None, **kw):
    x = x.detach().requires_grad_()
    loss = ops.cross_entropy(x, t, reduction=reduction, **kw)
    gout = torch.ones_like(loss) if gout is None else gout
    return loss.detach(), torch.autograd.grad(loss, x, gout)[0]


def _check_loss(got, want, dtype, gout):
    loss, grad = got
    # a row: exp of a product rounded once, summed, logarithm, two additions of
    # values below 32: 2^-24 * (32 + 32 + 16); sums of rows are fp64
    assert loss.dtype == torch.float32
    err = (loss.double().cpu() - want[0]).abs()
    assert (err <= 2.0 ** -24 * (80 + want[0].abs())
            * (loss.numel() == 1 and 64 or 1)).all(), float(err.max())
    # a gradient: probability off by 2^-24 * 32 of itself, one rounding; fp16's
    # steps end at 2^-24
    g = gout.double().cpu().abs().max()
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    err = (grad.double().cpu() - want[1]).abs()
    assert (err <= HALF[dtype] * 1.01 * want[1].abs() + 2.0 ** -18 * g * want[1].abs().clamp(max=1)
            + 2.0 ** -23 * g + tiny).all(), float(err.max())


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("n,v", SIZES)
def test_loss(n, v, reduction, dtype, device):
    x, t = _loss_inputs(n, v, dtype, device)
    got = _loss_and_grad(x, t, reduction)
    gout = torch.ones_like(got[0])
    _check_loss(got, loss_oracle(x, t, reduction, gout), dtype, gout)
    assert got[1].dtype == dtype and not got[1][t == -100].any()
    with torch.no_grad():
        assert torch.equal(ops.cross_entropy(x, t, reduction=reduction), got[0])


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_loss_factors(device):
    """What comes back multiplies the gradient before it is rounded: a loss
    scale keeps fp16 gradients in range, one value a row reaches its row."""
    x, t = _loss_inputs(40, 300, torch.float16, device)
    scale = torch.tensor(65536.0, device=device)
    _, grad = _loss_and_grad(x, t, "mean", scale)
    want = loss_oracle(x, t, "mean", scale)[1]
    err = (grad.double().cpu() - want).abs()
    assert (err <= 2.0 ** -11 * 1.01 * want.abs() + 2.0 ** -16 * want.abs() + 2.0 ** -7).all()
    each = torch.rand(40, device=device)
    got = _loss_and_grad(x.float(), t, "none", each)
    want = loss_oracle(x, t, "none", each)
    _check_loss(got, want, torch.float32, each)
    got = _loss_and_grad(x.float(), t, "none", torch.ones((), device=device).expand(40))
    assert torch.equal(got[1], _loss_and_grad(x.float(), t, "sum")[1])


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("v", [37, 9001])
def test_loss_edges(v, device):
    x = torch.randn(7, v).to(device)
    t = torch.tensor([0, 1, 2, 3, 4, 5, -1], device=device)
    x[0, 5:] = -math.inf          # a vocabulary shut off but for five
    x[1] = -math.inf              # nothing left
    x[2, 2] = -math.inf           # the label shut off
    x[3, 7] = math.nan
    x[4] = 3e38                   # far from zero, all alike
    t[5] = v                      # no such place, and another below zero
    loss, grad = _loss_and_grad(x, t, "none")
    assert torch.isfinite(loss[0]) and not grad[0, 5:].any()
    assert abs(float(grad[0].sum())) < 1e-6
    assert torch.isnan(loss[1])
    assert loss[2] == math.inf
    assert torch.isnan(loss[3]) and torch.isnan(grad[3]).any()
    assert abs(float(loss[4]) - math.log(v)) < 1e-5
    assert torch.isnan(loss[5]) and torch.isnan(grad[5]).all()
    assert torch.isnan(loss[6]) and torch.isnan(grad[6]).all()
    loss, grad = _loss_and_grad(x, t.fill_(-100), "mean")
    assert torch.isnan(loss) and not grad.any()
    loss, grad = _loss_and_grad(x, t, "sum")
    assert loss == 0 and not grad.any()
    assert float(ops.cross_entropy(x[:0], t[:0], reduction="sum")) == 0
    assert ops.cross_entropy(x[:0], t[:0], reduction="none").shape == (0,)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_loss_views(dtype, device):
    """Rows of a wider buffer, an odd start, transposed, other label types."""
    wide, t = _loss_inputs(12, 1000, dtype, device)
    t = t.clamp(max=900)
    for x in (wide[:, :901], wide[:, 3:904], wide[::2, :901], wide[1:, :901],
              wide[:, :901].t().contiguous().t()):
        n = x.shape[0]
        got = _loss_and_grad(x, t[:n].int(), "mean")
        want = _loss_and_grad(x.clone(memory_format=torch.contiguous_format), t[:n], "mean")
        assert abs(float(got[0] - want[0])) <= 2.0 ** -20 * float(want[0])
        torch.testing.assert_close(got[1], want[1], rtol=2 * HALF[dtype], atol=2.0 ** -24)
    other = t.masked_fill(t == -100, 0)
    a = _loss_and_grad(wide[:, :901], other, "mean", ignore_index=0)
    b = _loss_and_grad(wide[:, :901], other.masked_fill(other == 0, -100), "mean")
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_loss_of_no_rows_and_of_one_row_repeated(reduction, device):
    none = torch.zeros(0, 9, device=device, requires_grad=True)
    loss = ops.cross_entropy(none, torch.zeros(0, dtype=torch.int64, device=device),
                             reduction=reduction)
    loss.backward(torch.ones_like(loss))
    assert none.grad.shape == (0, 9) and loss.numel() == (reduction != "none")
    row = torch.randn(1, 901).to(device).requires_grad_()
    t = torch.tensor([3, 900, -100, 0, 3], device=device)
    loss = ops.cross_entropy(row.expand(5, 901), t, reduction=reduction)
    loss.backward(torch.ones_like(loss))
    want, grad = loss_oracle(row.expand(5, 901), t, reduction, torch.ones_like(loss))
    # five rows' gradients, and their sum, each within a few steps of values below 1
    assert ((row.grad.double().cpu()[0] - grad.sum(0)).abs() <= 5 * 2.0 ** -18).all()
    assert ((loss.double().cpu() - want).abs() <= 2.0 ** -18 * (1 + want.abs())).all()


@gpu
@pytest.mark.parametrize("lens", [[300, 40], [1500, 40, 700]])
def test_ops_gpu_from_two_threads(lens):
    """Each on a stream of its own, forward and backward."""
    steps = 20
    starts = torch.tensor(_starts(lens), dtype=torch.int32, device="cuda")
    data = [_inputs(lens, (4, 2), 64, seed=i, device="cuda") for i in range(2)]
    logits = [_loss_inputs(50, 9001, torch.bfloat16, "cuda", seed=i) for i in range(2)]
    want = [(_attend(*d, starts), _loss_and_grad(*x, "mean")) for d, x in zip(data, logits)]
    torch.cuda.synchronize()

    def work(i):
        out = []
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(steps):
                out.append((_attend(*data[i], starts), _loss_and_grad(*logits[i], "mean")))
            torch.cuda.current_stream().synchronize()
        return out

    with ThreadPoolExecutor(2) as pool:
        for i, got in enumerate(pool.map(work, range(2))):
            for attended, loss in got:
                assert all(torch.equal(x, y) for x, y in zip(attended, want[i][0]))
                assert all(torch.equal(x, y) for x, y in zip(loss, want[i][1]))


@gpu
def test_loss_gpu_more_rows_than_one_grid_counts():
    n = (1 << 26) + 37
    x = torch.zeros(n, 2, dtype=torch.float16, device="cuda")
    t = torch.ones(n, dtype=torch.int64, device="cuda")
    x[-1, 0] = 1.0
    loss, grad = _loss_and_grad(x, t, "sum")
    want = (n - 1) * math.log(2) + math.log(1 + math.e)
    assert abs(float(loss) / want - 1) <= 2.0 ** -22
    assert (grad[:-1, 0] == 0.5).all() and (grad[:-1, 1] == -0.5).all()
    p = 1 / (1 + math.exp(-1))
    assert abs(float(grad[-1, 0]) - p) <= 2.0 ** -11 and abs(float(grad[-1, 1]) + p) <= 2.0 ** -11


@gpu
def test_loss_gpu_captured():
    x, t = _loss_inputs(50, 4099, torch.bfloat16, "cuda")
    x.requires_grad_()

    def step():
        loss = ops.cross_entropy(x, t)
        return loss, torch.autograd.grad(loss, x)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for seed in range(1, 4):
        y, u = _loss_inputs(50, 4099, torch.bfloat16, "cuda", seed=seed)
        with torch.no_grad():
            x.copy_(y)
            t.copy_(u)
        graph.replay()
        got = [z.detach().clone() for z in static]
        want = _loss_and_grad(y, u, "mean")
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        torch.cuda.synchronize()


def test_loss_agrees_with_torch():
    x, t = _loss_inputs(20, 33, torch.float32, "cpu")
    torch.testing.assert_close(ops.cross_entropy(x, t), torch.nn.functional.cross_entropy(x, t))
    x = x[:4].double().requires_grad_()
    assert torch.autograd.gradcheck(lambda y: ops.cross_entropy(y, t[:4]), x)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_loss_refuses(device):
    x, t = _loss_inputs(4, 9, torch.float32, device)
    for args in ((x[0], t), (x, t[:3]), (x, t.float()), (x[None], t[None]), (x[:, :0], t)):
        with pytest.raises(ValueError):
            ops.cross_entropy(*args)
    with pytest.raises(ValueError):
        ops.cross_entropy(x, t, reduction="max")
    if device == "cuda":
        with pytest.raises(ValueError):
            ops.cross_entropy(x.double(), t)
        with pytest.raises(ValueError):
            ops.cross_entropy(x, t.cpu())


# ------------------------------------------------------------- gradient norm

def _params(shapes, dtypes, device, std=0.1, seed=0):
    gen = torch.Generator().manual_seed(seed)
    out = []
    for i, shape in enumerate(shapes):
        dtype = dtypes[i % len(dtypes)]
        p = torch.nn.Parameter(torch.zeros(shape, dtype=dtype, device=device))
        p.grad = (torch.randn(shape, generator=gen) * std).to(dtype).to(device)
        out.append(p)
    return out


def _check_clip(params, limit):
    """Clips, and compares with 64 bits: the factor is rounded to fp32, the
    product to fp32 and to the gradient's type."""
    before = [p.grad.detach().double().cpu() for p in params]
    want = math.sqrt(sum(float(g.square().sum()) for g in before))
    assert abs(float(ops.grad_norm(params)) - want) <= 2.0 ** -23 * want
    norm = ops.clip_grad_norm_(params, limit)
    assert norm.dtype == torch.float32 and norm.dim() == 0
    assert abs(float(norm) - want) <= 2.0 ** -23 * want
    factor = min(1.0, limit / (want + 1e-6))
    for p, g in zip(params, before):
        got = p.grad.detach().double().cpu()
        if factor == 1.0:
            assert torch.equal(got, g)
            continue
        tiny = 2.0 ** -25 if p.dtype == torch.float16 else 0.0
        err = (got - g * factor).abs()
        assert (err <= (HALF[p.dtype] + 2.0 ** -22) * g.abs() * factor * 1.01 + tiny).all()


MIXED = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [(1,), (), (7, 3), (0,), (8192,), (8193,), (4095, 5), (3, 1, 2), (100_000,), (2,)]


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("dtypes", [MIXED[:1], MIXED[1:2], MIXED])
@pytest.mark.parametrize("limit", [0.0, 0.5, 1e6, math.inf])
def test_clip(limit, dtypes, device):
    _check_clip(_params(SHAPES, dtypes, device), limit)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_clip_many(device):
    """More tensors than one launch takes."""
    _check_clip(_params([(i % 37 + 1,) for i in range(300)], MIXED, device), 0.25)


@gpu
def test_clip_gpu_large():
    params = _params([(3_000_001,), (5, 700_003)], MIXED[:2], "cuda")
    _check_clip(params, 1.0)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_clip_strides_and_alignment(device):
    """Slices of one flat buffer at odd starts, turned and spaced tensors:
    nothing beside them changes."""
    for dtype in MIXED:
        flat = torch.randn(40_000).to(dtype).to(device)
        keep = flat.clone()
        cuts = [(1, 8), (9, 9001), (9002, 9003), (9011, 20_000)]
        params = []
        for a, b in cuts:
            p = torch.nn.Parameter(torch.zeros(b - a, dtype=dtype, device=device))
            p.grad = flat[a:b]
            params.append(p)
        p = torch.nn.Parameter(torch.zeros(30, 40, dtype=dtype, device=device))
        p.grad = torch.randn(40, 30).to(dtype).to(device).t()
        params.append(p)
        gaps = torch.randn(50, 20).to(dtype).to(device)
        was = gaps.clone()
        p = torch.nn.Parameter(torch.zeros(25, 10, dtype=dtype, device=device))
        p.grad = gaps[::2, 3:13]
        params.append(p)
        _check_clip(params, 0.5)
        inside = torch.zeros(40_000, dtype=torch.bool)
        for a, b in cuts:
            inside[a:b] = True
        assert torch.equal(flat.cpu()[~inside], keep.cpu()[~inside])
        assert torch.equal(gaps[1::2], was[1::2]) and torch.equal(gaps[:, 13:], was[:, 13:])
        assert torch.equal(gaps[:, :3], was[:, :3])


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_clip_range(device):
    """Squares that 32 bits do not hold."""
    for std in (1e25, 1e-30):
        params = _params([(500,)], MIXED[:1], device, std=std)
        want = float(params[0].grad.double().norm())
        assert abs(float(ops.grad_norm(params)) / want - 1) < 1e-6
    before = params[0].grad.clone()
    ops.clip_grad_norm_(params, 1.0)
    assert torch.equal(params[0].grad, before)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_clip_factor_below_the_smallest_normal_number(device):
    """1e-3 / 1e38 has few bits in fp32; the results, near 1e-4, have all."""
    params = _params([(500,), (8, 9)], MIXED[:2], device, std=3e36)
    _check_clip(params, 1e-3)
    assert 1e-6 < float(params[0].grad.abs().max()) < 1e-3


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_clip_refuses_shared_memory(device):
    one, two = _params([(4, 6), (4, 6)], MIXED[:1], device)
    both = torch.randn(4, 12, device=device)
    keep = both.clone()
    one.grad, two.grad = both[:, :6], both[:, 6:]
    for params in ([one, one], [one, two]):
        with pytest.raises(ValueError, match="share or interleave"):
            ops.clip_grad_norm_(params, 0.1)
    assert torch.equal(both, keep)
    norm = float(keep.double().square().sum().sqrt())
    assert abs(float(ops.grad_norm([one, two])) / norm - 1) < 1e-6
    one, two = _params([(2, 6), (2, 6)], MIXED[:1], device)
    one.grad, two.grad = both[:2, :6], both[2:, :6]     # one after the other is fine
    _check_clip([one, two], 0.1)
    assert torch.equal(both[:, 6:], keep[:, 6:])


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_clip_not_finite(device):
    """As torch's: an infinite norm leaves zeros and NaN, a NaN norm NaN."""
    for bad in (math.inf, math.nan):
        params = _params([(5,), (9000,)], MIXED[:1], device)
        params[1].grad[77] = bad
        twin = [p.grad.clone() for p in params]
        with pytest.raises(RuntimeError):
            ops.clip_grad_norm_(iter(params), 1.0, error_if_nonfinite=True)
        assert all(torch.equal(p.grad, t) or bad != bad for p, t in zip(params, twin))
        norm = ops.clip_grad_norm_(params, 1.0)
        other = [torch.nn.Parameter(torch.zeros_like(p)) for p in params]
        for q, t in zip(other, twin):
            q.grad = t
        torch.testing.assert_close(norm, torch.nn.utils.clip_grad_norm_(other, 1.0),
                                   equal_nan=True)
        for p, q in zip(params, other):
            assert torch.equal(torch.isnan(p.grad), torch.isnan(q.grad))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_clip_forms(device):
    one = torch.nn.Parameter(torch.zeros(3, device=device))
    assert float(ops.clip_grad_norm_(one, 1.0)) == 0.0     # no gradient
    assert float(ops.grad_norm([])) == 0.0
    one.grad = torch.tensor([3.0, 0.0, 4.0], device=device)
    version = one.grad._version
    assert float(ops.clip_grad_norm_((p for p in [one]), 1.0)) == 5.0
    assert one.grad._version > version
    torch.testing.assert_close(one.grad.cpu(), torch.tensor([0.6, 0.0, 0.8]))
    one.grad = torch.zeros(3, device=device)
    assert float(ops.clip_grad_norm_(one, 0.0)) == 0.0
    none = torch.nn.Parameter(torch.zeros(0, device=device))
    none.grad = torch.zeros(0, device=device)
    assert float(ops.clip_grad_norm_(none, 1.0)) == 0.0


@gpu
def test_clip_gpu_captured():
    """The norm and whether it clips are of each replay's own gradients."""
    params = _params([(300, 7), (9001,)], MIXED, "cuda")
    twins = _params([(300, 7), (9001,)], MIXED, "cuda")
    ops.clip_grad_norm_(params, 1.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = ops.clip_grad_norm_(params, 1.0)
    for std in (0.1, 1e-4, 3.0):
        new = _params([(300, 7), (9001,)], MIXED, "cuda", std=std)
        for p, q, n in zip(params, twins, new):
            p.grad.copy_(n.grad)
            q.grad.copy_(n.grad)
        graph.replay()
        want = ops.clip_grad_norm_(twins, 1.0)
        assert torch.equal(norm, want)
        assert all(torch.equal(p.grad, q.grad) for p, q in zip(params, twins))
        torch.cuda.synchronize()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_clip_refuses(device):
    params = _params([(4,), (5,)], MIXED[:1], device)
    for limit in (-1.0, math.nan):
        with pytest.raises(ValueError):
            ops.clip_grad_norm_(params, limit)
    wide = torch.nn.Parameter(torch.zeros(4, dtype=torch.float64, device=device))
    wide.grad = torch.ones_like(wide)
    with pytest.raises(ValueError):
        ops.clip_grad_norm_([wide], 1.0)
    if device == "cuda":
        with pytest.raises(ValueError):
            ops.clip_grad_norm_([params[0], params[0]], 1.0)
        spread = torch.nn.Parameter(torch.zeros(4, device=device))
        spread.grad = torch.ones(1, device=device).expand(4)
        with pytest.raises(ValueError):
            ops.clip_grad_norm_([spread], 1.0)
        assert float(ops.grad_norm([spread])) == 2.0
        host = torch.nn.Parameter(torch.zeros(4))
        host.grad = torch.ones(4)
        with pytest.raises(ValueError):
            ops.clip_grad_norm_([params[0], host], 1.0)
        assert torch.equal(host.grad, torch.ones(4))


@gpu
def test_second_derivatives_refused_gpu():
    q, k, v, _ = _inputs([20], (2, 1), 64, device="cuda")
    q.requires_grad_()
    out = ops.packed_attention(q, k, v, torch.tensor([0, 20], device="cuda"))
    dq, = torch.autograd.grad(out.float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        dq.float().sum().backward()
    x, t = _loss_inputs(4, 9, torch.float32, "cuda")
    dx, = torch.autograd.grad(ops.cross_entropy(x.requires_grad_(), t), x, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        dx.sum().backward()


@gpu
def test_attention_gpu_part_of_the_gradients():
    q, k, v, dout = _inputs([90], (4, 2), 64, device="cuda")
    starts = torch.tensor([0, 90], device="cuda")
    want = _attend(q, k, v, dout, starts)[1:]
    for ask in ([0], [1], [2], [0, 2]):
        parts = [x.detach().requires_grad_(i in ask) for i, x in enumerate((q, k, v))]
        out = ops.packed_attention(*parts, starts)
        got = torch.autograd.grad(out, [parts[i] for i in ask], dout)
        assert all(torch.equal(g, want[i]) for g, i in zip(got, ask))


# -------------------------------------------------------------- all together

def test_pack_samples():
    from runbookai_amd.engine.train import pack_samples

    ids, starts, targets = pack_samples([([5, 6, 7, 8], 2), ([], 0), ([9], 0), ([1, 2], 1)])
    assert ids.tolist() == [5, 6, 7, 8, 9, 1, 2]
    assert starts.tolist() == [0, 4, 4, 5, 7]
    assert targets.tolist() == [-100, 7, 8, -100, -100, 2, -100]


def test_packed_model_agrees_with_padded():
    """Logits and gradients of a packed batch are those of each sequence by
    itself; both in fp32, whose sums differ in order only."""
    from runbookai_amd.engine.train import CONFIGS, TrainableLlama, pack_samples

    torch.manual_seed(0)
    model = TrainableLlama(CONFIGS["tiny"])
    gen = torch.Generator().manual_seed(1)
    samples = [(torch.randint(0, 4096, (n,), generator=gen).tolist(), n // 2) for n in (7, 1, 12)]
    ids, starts, targets = pack_samples(samples)
    ops.cross_entropy(model.forward_packed(ids, starts), targets).backward()
    packed = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad()
    logits, labels = [], []
    for tokens, answer in samples:
        logits.append(model(torch.tensor(tokens)[None])[0])
        t = torch.tensor(tokens[1:] + [-100])
        t[:max(0, answer - 1)] = -100
        labels.append(t)
    torch.testing.assert_close(model.forward_packed(ids, starts), torch.cat(logits),
                               rtol=1e-4, atol=1e-5)
    torch.nn.functional.cross_entropy(torch.cat(logits), torch.cat(labels)).backward()
    for n, p in model.named_parameters():
        torch.testing.assert_close(packed[n], p.grad, rtol=1e-3, atol=1e-6, msg=n)


def test_packed_model_refuses():
    from runbookai_amd.engine.train import CONFIGS, TrainableLlama

    model = TrainableLlama(CONFIGS["tiny"])
    ids = torch.zeros(10, dtype=torch.long)
    for starts in ([0, 11], [0, 4, 3], [-1, 10], []):
        with pytest.raises(ValueError):
            model.forward_packed(ids, torch.tensor(starts, dtype=torch.int32))
    with pytest.raises(ValueError):
        model.forward_packed(ids[None], torch.tensor([0, 10]))
    with pytest.raises(ValueError):
        model.forward_packed(torch.zeros(5000, dtype=torch.long), torch.tensor([0, 5000]))
    assert model.forward_packed(ids[:0], torch.tensor([0])).shape == (0, 4096)


def test_packed_training_script_runs(tmp_path):
    import subprocess
    import sys

    proc = subprocess.run(
        [sys.executable, "scripts/train_policy.py", "--cases", "4", "--steps", "2", "--out",
         str(tmp_path), "--max-len", "768", "--batch-tokens", "2048", "--packed"],
        capture_output=True, text=True, timeout=600)
    assert proc.returncode == 0, proc.stderr[-1500:]
    assert (tmp_path / "model.safetensors").exists()


@gpu
def test_training_step_gpu():
    """Attention, loss and clipping as a step runs them; each stage is held to
    64 bits on what the stage before gave it."""
    lens, hq, hk, d, vocab = [150, 0, 1, 200], 4, 2, 64, 1000
    q, k, v, _ = _inputs(lens, (hq, hk), d, pad=9, device="cuda")
    starts = _starts(lens)
    T = q.shape[0]
    gen = torch.Generator().manual_seed(5)
    w = torch.nn.Parameter((torch.randn(vocab, hq * d, generator=gen) * 0.05).cuda())
    targets = torch.randint(0, vocab, (T,), generator=gen).cuda()
    targets[::3] = -100
    targets[starts[-1]:] = -100
    parts = [torch.nn.Parameter(x) for x in (q, k, v)]
    out = ops.packed_attention(*parts, torch.tensor(starts, device="cuda"))
    out.retain_grad()
    logits = out.reshape(T, -1).float() @ w.t()
    logits.retain_grad()
    loss = ops.cross_entropy(logits, targets)
    loss.backward()
    one = torch.ones((), device="cuda")
    _check_loss((loss.detach(), logits.grad), loss_oracle(logits, targets, "mean", one),
                torch.float32, one)
    want, tol = attention_oracle(q, k, v, out.grad, starts, 1 / math.sqrt(d))
    _within([out.detach()] + [p.grad for p in parts], want, tol)
    _check_clip(parts + [w], 0.01)


@gpu
def test_packed_model_gpu():
    """The policy's forward and backward pass under autocast, against fp32 on
    the host. A row passes some 16 roundings to bf16 on its way to a logit."""
    from runbookai_amd.engine.train import CONFIGS, TrainableLlama, pack_samples

    torch.manual_seed(0)
    model = TrainableLlama(CONFIGS["tiny"])
    gen = torch.Generator().manual_seed(1)
    samples = [(torch.randint(0, 4096, (n,), generator=gen).tolist(), n // 3)
               for n in (200, 3, 1, 333, 64)]
    ids, starts, targets = pack_samples(samples)
    want = model.forward_packed(ids, starts)
    want_loss = ops.cross_entropy(want, targets)
    model = model.cuda()
    with torch.autocast(device_type="cuda", dtype=torch.bfloat16):
        got = model.forward_packed(ids.cuda(), starts)
    loss = ops.cross_entropy(got, targets.cuda())
    slack = 16 * H * float(want.detach().abs().max())
    assert (got.detach().float().cpu() - want.detach()).abs().max() <= slack
    assert abs(float(loss.detach()) - float(want_loss.detach())) <= slack
    loss.backward()
    norm = ops.clip_grad_norm_(model.parameters(), 0.5, error_if_nonfinite=True)
    assert float(norm) > 0
    assert float(ops.grad_norm(model.parameters())) <= 0.5 * (1 + 1e-5)


# ------------------------------------------- tensors that are more than memory

def test_ops_refuse_tensors_without_memory():
    """Fake tensors have a shape and a device and no memory behind them."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        q = torch.empty(4, 2, 64, dtype=torch.bfloat16, device="cuda")
        starts = torch.empty(2, dtype=torch.int32, device="cuda")
        logits = torch.empty(4, 9, device="cuda")
        targets = torch.empty(4, dtype=torch.int64, device="cuda")
        p = torch.nn.Parameter(torch.empty(5, device="cuda"))
        p.grad = torch.empty(5, device="cuda")
        for call in (lambda: ops.packed_attention(q, q, q, starts),
                     lambda: ops.packed_attention(q.requires_grad_(), q, q, starts),
                     lambda: ops.cross_entropy(logits, targets),
                     lambda: ops.grad_norm([p]), lambda: ops.clip_grad_norm_([p], 1.0)):
            with pytest.raises(ValueError, match="plain tensor"):
                call()


@gpu
def test_ops_gpu_refuse_freed_memory():
    """A parameter whose storage was let go until it is needed again."""
    q, k, v, _ = _inputs([4], (4, 2), 64, device="cuda")
    starts = torch.tensor([0, 4], device="cuda")
    k.untyped_storage().resize_(0)
    with pytest.raises(ValueError, match="plain tensor"):
        ops.packed_attention(q, k, v, starts)
    p = torch.nn.Parameter(torch.zeros(5, device="cuda"))
    p.grad = torch.ones(5, device="cuda")
    p.grad.untyped_storage().resize_(0)
    for call in (lambda: ops.grad_norm([p]), lambda: ops.clip_grad_norm_([p], 1.0)):
        with pytest.raises(ValueError, match="plain tensor"):
            call()


@gpu
def test_ops_gpu_refuse_results_without_memory():
    """Real inputs while a mode makes every new tensor a fake one."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    q, k, v, _ = _inputs([4], (4, 2), 64, device="cuda")
    x, t = _loss_inputs(4, 9, torch.float32, "cuda")
    p = torch.nn.Parameter(torch.zeros(5, device="cuda"))
    p.grad = torch.ones(5, device="cuda")
    rows = x.detach().requires_grad_()
    loss = ops.cross_entropy(rows, t)
    one = torch.ones_like(loss)
    for kind in (torch.int32, torch.int64):
        starts = torch.tensor([0, 4], dtype=kind, device="cuda")
        leaf = q.detach().requires_grad_()
        out = ops.packed_attention(leaf, k, v, starts)
        with FakeTensorMode(allow_non_fake_inputs=True):
            for call in (lambda: ops.packed_attention(q, k, v, starts),
                         lambda: ops.packed_attention(leaf, k, v, starts),
                         lambda: torch.autograd.grad(out, leaf, q, retain_graph=True),
                         lambda: torch.autograd.grad(loss, rows, one, retain_graph=True),
                         lambda: ops.cross_entropy(x, t), lambda: ops.grad_norm([p]),
                         lambda: ops.clip_grad_norm_([p], 1.0)):
                with pytest.raises(ValueError, match="plain tensor"):
                    call()
    assert (p.grad == 1).all()


def _tangents(device):
    """Outputs' tangents for tangents of one input each, and of a gradient."""
    import torch.autograd.forward_ad as fwd

    dtype = torch.bfloat16 if device == "cuda" else torch.float64
    q, k, v, dout = _inputs([7, 2], (2, 1), 64, device=device, dtype=dtype)
    starts = torch.tensor([0, 7, 9], device=device)
    x, t = _loss_inputs(4, 9, torch.float32, device)
    way = torch.ones_like
    with fwd.dual_level():
        def tangent(call):
            return lambda: fwd.unpack_dual(call()).tangent

        yield tangent(lambda: ops.packed_attention(fwd.make_dual(q, way(q)), k, v, starts))
        yield tangent(lambda: ops.packed_attention(q, fwd.make_dual(k, way(k)), v, starts))
        yield tangent(lambda: ops.packed_attention(q, k, fwd.make_dual(v, way(v)), starts))
        yield tangent(lambda: ops.cross_entropy(fwd.make_dual(x, way(x)), t))
        leaf = v.detach().requires_grad_()
        yield tangent(lambda: torch.autograd.grad(ops.packed_attention(q, k, leaf, starts), leaf,
                                                  fwd.make_dual(dout, way(dout)))[0])
        rows = x.detach().requires_grad_()
        yield tangent(lambda: torch.autograd.grad(ops.cross_entropy(rows, t), rows,
                                                  fwd.make_dual(x.new_ones(()), x.new_ones(())))[0])
        p = torch.nn.Parameter(torch.zeros_like(x))
        p.grad = fwd.make_dual(x, way(x))
        yield tangent(lambda: ops.grad_norm([p]))


def test_forward_mode_derivatives():
    """On the host every op carries tangents."""
    for call in _tangents("cpu"):
        assert call() is not None


@gpu
def test_forward_mode_derivatives_refused_gpu():
    """The kernels do not, and must not return an output that looks constant."""
    for call in _tangents("cuda"):
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call()


@gpu
def test_trace_refused_gpu():
    """A recorded trace would hold the output's allocation and no kernel."""
    q, k, v, _ = _inputs([9], (4, 2), 64, device="cuda")
    starts = torch.tensor([0, 9], device="cuda")
    x, t = _loss_inputs(4, 9, torch.float32, "cuda")
    for call, args in ((lambda q: ops.packed_attention(q, k, v, starts), (q,)),
                       (lambda x: ops.cross_entropy(x, t), (x,))):
        with pytest.raises(NotImplementedError, match="trace"):
            torch.jit.trace(call, args, check_trace=False)
    for call in (lambda: torch.func.grad(lambda q: ops.packed_attention(q, k, v, starts).sum())(q),
                 lambda: torch.func.vmap(lambda x: ops.cross_entropy(x, t))(x[None])):
        with pytest.raises((RuntimeError, ValueError)):   # wrappers without memory
            call()


# ----------------------------------------------------------- how work is split

@gpu
@pytest.mark.parametrize("empty", [0, 62])   # tiles from a search, from a table
@pytest.mark.parametrize("d", [64, 128])
def test_attention_gpu_unused_rows_change_no_split(d, empty):
    """Where dk and dv are summed by several workgroups the split shows in their
    last bits: a sequence in a buffer of several times its length is split as
    by itself. The buffer's length chooses a plan too; here it is the same one:
    at most 7000 / 128 + 63 + 2 = 119 tiles, times 4 heads below the 512 up to
    which two teams take a tile, times 2 heads (and 2 halves at d 64) below the
    256 (768) up to which four parts do."""
    heads = (4, 2)
    n, T = 1500, 7000
    q, k, v, dout = _inputs([n], heads, d, device="cuda")
    starts = torch.tensor([0] * (empty + 1) + [n], dtype=torch.int32, device="cuda")
    want = _attend(q, k, v, dout, starts)
    for before in (0, 4000):
        wide = [torch.zeros(T, *x.shape[1:], dtype=x.dtype, device="cuda")
                for x in (q, k, v, dout)]
        for x, y in zip(wide, (q, k, v, dout)):
            x[before:before + n] = y
        for x, y in zip(_attend(*wide, starts + before), want):
            assert torch.equal(x[before:before + n], y)
            assert not x[:before].any() and not x[before + n:].any()


@gpu
@pytest.mark.parametrize("lens,heads,d,parts", [
    ([37], (32, 8), 128, 0), ([1] * 93, (32, 8), 128, 0), ([12] * 58, (64, 8), 128, 2),
    ([1] * 30, (64, 1), 64, 4), ([100, 7], (64, 2), 128, 4), ([1500, 40, 700], (8, 2), 128, 4)])
def test_attention_gpu_scratch_goes_by_rows(lens, heads, d, parts):
    """A backward pass takes what it returns, an fp32 number a row and head, and
    an fp32 copy of dk and dv for each part (none where nothing can be long
    enough for one), whatever the number of sequences."""
    q, k, v, dout = _inputs(lens, heads, d, pad=5, device="cuda")
    starts = torch.tensor(_starts(lens), dtype=torch.int32, device="cuda")
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = ops.packed_attention(*leaves, starts)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = torch.autograd.grad(out, leaves, dout)
    took = torch.cuda.max_memory_allocated() - before
    pair = k.numel() + v.numel()
    most = 2 * (q.numel() + pair) + 4 * q.shape[0] * heads[0] + 4 * parts * pair
    # and 4 bytes each of at most 3 * 768 counters, and every allocation's end
    assert took <= most + 2 ** 16, (took, most)
    want, tol = attention_oracle(q, k, v, dout, _starts(lens), 1.0 / math.sqrt(d))
    _within(got, want[1:], tol[1:])


# ------------------------------------------------- where a clipping call runs

@gpu
@pytest.mark.parametrize("frozen,device", [("cpu", "cuda"), ("cuda", "cpu"), ("cuda", "cuda")])
def test_clip_gpu_frozen_parameters_decide_nothing(frozen, device, monkeypatch):
    """Parameters without a gradient are passed over, the first one too: GPU
    gradients go to the kernels, host gradients to the host's path."""
    if device == "cuda":
        monkeypatch.setattr(reference, "grad_norm", None)
        monkeypatch.setattr(reference, "grad_clip", None)
    shut = torch.nn.Parameter(torch.zeros(7, device=frozen), requires_grad=False)
    params = _params([(500,), (3, 4)], MIXED[:1], device)
    for order in ([shut] + params, params + [shut]):
        assert ops.grad_norm(order).device.type == device
        norm = float(torch.cat([p.grad.double().flatten() for p in params]).norm())
        assert abs(float(ops.clip_grad_norm_(order, 0.25)) - norm) <= 2.0 ** -23 * norm
        assert ops.clip_grad_norm_(order, 0.25, error_if_nonfinite=True).device.type == device
        assert float(ops.grad_norm(order)) <= 0.25 * (1 + 2.0 ** -22)
        for p in params:
            p.grad.mul_(8.0)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_clip_without_gradients_stays_on_the_device(device):
    params = [torch.nn.Parameter(torch.zeros(3, device=device)) for _ in range(2)]
    for norm in (ops.grad_norm(params), ops.clip_grad_norm_(params, 1.0),
                 ops.clip_grad_norm_(params, 1.0, error_if_nonfinite=True)):
        assert norm.device.type == device and norm.dtype == torch.float32 and float(norm) == 0.0
    assert float(ops.clip_grad_norm_([], 1.0)) == 0.0


# ------------------------------------------------------------ scales at the end

@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_attention_scales_at_the_ends(device):
    """A scale that fp32 rounds to 0 (or to fewer bits) is refused; with the
    smallest that it holds a row's probabilities are all alike, and its rows
    are means of the values so far."""
    q, k, v, dout = _inputs([40], (4, 2), 64, device=device)
    starts = torch.tensor([0, 40], device=device)
    for scale in (1e-46, 1e-300, 2.0 ** -149, 2.0 ** -127):
        with pytest.raises(ValueError, match="scale"):
            ops.packed_attention(q, k, v, starts, scale=scale)
    for scale in (2.0 ** -126, 1e-30):
        got = _attend(q, k, v, dout, starts, scale)
        want, tol = attention_oracle(q, k, v, dout, [0, 40], scale)
        # dq and dk are near the smallest numbers that bf16 holds, or below
        _within([got[0], got[3]], [want[0], want[3]], [tol[0], tol[3]], ("out", "dv"))
        assert all(torch.isfinite(x).all() for x in got)


# ------------------------------------------------------ logits that are views

@gpu
@pytest.mark.parametrize("dtype", MIXED)
@pytest.mark.parametrize("n,width,cols", [
    (256, 1009, slice(0, 1001)), (256, 1001, slice(1, None)), (200, 1003, slice(1, 1000)),
    (24, 9003, slice(0, 9001)), (24, 9001, slice(3, None)), (300, 5, slice(1, 4))])
def test_loss_gpu_views_are_not_copied(n, width, cols, dtype):
    """Columns of a wider buffer, at every distance to a 16-byte boundary: the
    backward pass takes its result's memory and no copy of the logits."""
    wide, t = _loss_inputs(n + 1, width, dtype, "cuda")
    x, t = wide[1:, cols], t[1:].clone()
    t[t >= x.shape[1]] = 0
    x = x.detach().requires_grad_()
    loss = ops.cross_entropy(x, t)
    one = torch.ones_like(loss)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    grad, = torch.autograd.grad(loss, x, one)
    took = torch.cuda.max_memory_allocated() - before
    assert took <= grad.numel() * grad.element_size() + 512
    _check_loss((loss.detach(), grad), loss_oracle(x, t, "mean", one), dtype, one)


@gpu
@pytest.mark.parametrize("starts", [[0, 5], [-1, 4], [0, 3, 2, 4]])
def test_attention_on_the_host_checks_starts_of_the_gpu(starts):
    q, k, v, _ = _inputs([4], (4, 2), 64)
    with pytest.raises(ValueError):
        ops.packed_attention(q, k, v, torch.tensor(starts, device="cuda"))
    fine = torch.tensor([0, 3, 4])
    assert torch.equal(ops.packed_attention(q, k, v, fine.cuda()),
                       ops.packed_attention(q, k, v, fine))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.complex64])
def test_ops_refuse_other_numbers(dtype, device):
    """A probability is no whole number."""
    q, k, v, _ = _inputs([4], (4, 2), 64, device=device)
    starts = torch.tensor([0, 4], device=device)
    with pytest.raises(ValueError):
        ops.packed_attention(q.to(dtype), k.to(dtype), v.to(dtype), starts)
    x, t = _loss_inputs(4, 9, torch.float32, device)
    with pytest.raises(ValueError):
        ops.cross_entropy(x.to(dtype), t)


@gpu
def test_attention_gpu_refuses_more_heads_than_one_grid_counts():
    """3 tiles are rounded up to the 8 XCDs that share a kv head: with 2.7
    million query heads that is more than 2^32 threads."""
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device="cuda")
    q = x.expand(1, 2_700_000, 64)
    starts = torch.tensor([0, 1], device="cuda")
    with pytest.raises(RuntimeError, match="too many rows, sequences and heads"):
        ops.packed_attention(q, x, x, starts)
    got = ops.packed_attention(q[:, :100_000], x + 1, x + 1, starts)
    assert (got == 1).all()


# ------------------------------------------------------------- closer bounds

@gpu
@pytest.mark.parametrize("n,v", [(1, 1), (1, 777), (1, 9001), (3, 4099), (999, 33), (40_000, 9),
                                 (300, 9001), (100_001, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_loss_gpu_sums_of_rows_are_rounded_once(n, v, dtype):
    """The rows' losses, each as a loss of its own, added in 64 bits: a sum and
    a mean are within half a step of fp32 (and what 64 bits round)."""
    x, t = _loss_inputs(n, v, dtype, "cuda", labelled=0.9)
    rows = ops.cross_entropy(x, t, reduction="none").double().cpu()
    want = loss_oracle(x, t, "none", torch.ones(n))[0]
    # exp of a product rounded once, summed, logarithm, two additions: as _check_loss
    assert ((rows - want).abs() <= 2.0 ** -24 * (80 + want)).all()
    for reduction, exact in (("sum", rows.sum()), ("mean", rows.sum() / (t != -100).sum().cpu())):
        got = ops.cross_entropy(x, t, reduction=reduction).double().cpu()
        assert (got - exact).abs() <= 2.0 ** -24 * (1 + 2.0 ** -20) * exact.abs()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_clip_leaves_gradients_whose_norm_is_not_finite(bad, device):
    params = _params([(5,), (9000,)], MIXED[:1], device)
    params[1].grad[77] = bad
    before = [p.grad.clone() for p in params]
    with pytest.raises(RuntimeError):
        ops.clip_grad_norm_(params, 1.0, error_if_nonfinite=True)
    for p, g in zip(params, before):
        torch.testing.assert_close(p.grad, g, rtol=0, atol=0, equal_nan=True)
    assert torch.isfinite(params[0].grad).all() and params[0].grad.any()


# ------------------------------------------------------------ every plan of dk, dv

@gpu
@pytest.mark.parametrize("lens,heads,d,parts", [
    # in up to two parts, and split: more workgroups than run at once
    ([0] * 25 + [1500], (32, 8), 128, 2), ([0] * 4 + [1500, 130], (64, 16), 128, 2),
    ([0] * 50 + [1500], (16, 8), 64, 2), ([0] * 70 + [100, 1400], (16, 8), 64, 2),
    # in one: more than three times as many
    ([0] * 25 + [300, 1], (32, 32), 128, 1), ([0] * 32 + [500], (32, 32), 64, 1),
    ([0] * 150 + [1100, 60], (32, 8), 64, 1), ([0] * 90 + [1100, 60], (32, 8), 128, 1)])
def test_attention_gpu_plans_of_parts(lens, heads, d, parts):
    """Which plan it is shows in the memory: a copy of dk and dv in fp32 a part,
    where there are several."""
    q, k, v, dout = _inputs(lens, heads, d, pad=5, device="cuda")
    starts = torch.tensor(_starts(lens), dtype=torch.int32, device="cuda")
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = ops.packed_attention(*leaves, starts)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = torch.autograd.grad(out, leaves, dout)
    took = torch.cuda.max_memory_allocated() - before
    pair = k.numel() + v.numel()
    rest = 2 * (q.numel() + pair) + 4 * q.shape[0] * heads[0]
    # allocations end at 2 MiB at most behind what was asked for
    copies = (took - rest) / (4 * pair)
    assert round(copies) == (parts if parts > 1 else 0), copies
    want, tol = attention_oracle(q, k, v, dout, _starts(lens), 1.0 / math.sqrt(d))
    _within((out.detach(), *got), want, tol)
    for _ in range(5):
        for x, y in zip(_attend(q, k, v, dout, starts)[1:], got):
            assert torch.equal(x, y)


@gpu
def test_attention_gpu_coarse_table():
    """From 524288 rows on the table sorts tiles by two of their numbers at once:
    the same bits as batches of a quarter each (which have the same plan: over
    512 workgroups for out and dq, over 2304 for dk and dv), and some sequences
    held to 64 bits."""
    gen = torch.Generator().manual_seed(7)
    quarters = []
    for _ in range(4):
        lens = torch.randint(0, 1500, (150,), generator=gen).tolist()
        quarters.append(lens + [150_000 - sum(lens)])
    d, heads = 64, (2, 1)
    lens = sum(quarters, [])
    q, k, v, dout = _inputs(lens, heads, d, device="cuda")
    assert q.shape[0] == 600_000
    starts = _starts(lens)
    got = _attend(q, k, v, dout, torch.tensor(starts, dtype=torch.int32, device="cuda"))
    for i, quarter in enumerate(quarters):
        a, b = i * 150_000, (i + 1) * 150_000
        part = _attend(q[a:b], k[a:b], v[a:b], dout[a:b],
                       torch.tensor(_starts(quarter), dtype=torch.int32, device="cuda"))
        assert all(torch.equal(x[a:b], y) for x, y in zip(got, part))
    for i in (0, 1, 200, len(lens) - 3):
        a, b = starts[i], starts[i + 1]
        want, tol = attention_oracle(*(x[a:b] for x in (q, k, v, dout)), [0, b - a],
                                     1.0 / math.sqrt(d))
        _within([x[a:b] for x in got], want, tol)
