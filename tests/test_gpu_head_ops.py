"""The head's operators on the GPU against their definitions in 64 bits: cross entropy and its
gradients, rows to 8-bit integers, the product of such rows.

Tolerances are worst-case bounds computed for each output entry from the inputs: u is half a step of the
16-bit type, E24 = 2^-24 that of fp32.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E24 = 2.0 ** -24
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# smallest step of the type's numbers near zero (half of it is what a rounding can lose there)
TINY = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
IGNORE = -100


@pytest.fixture(scope="module")
def ext():
    import qwen_megakernel_C

    return qwen_megakernel_C


def make(tokens, vocab, width, dtype, seed=0, lean=8.0, pad=0):
    """Hidden rows that lean towards their targets, the head's rows, targets; rows `pad` apart."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rows(n, std):
        t = torch.randn(n, width + pad, device="cuda", generator=g).mul_(std).to(dtype)
        return t[:, :width]

    w = rows(vocab, 1.2 / math.sqrt(width))
    y = torch.randint(0, vocab, (tokens,), device="cuda", generator=g)
    h = rows(tokens, 1.0)
    h += (lean * torch.rand(tokens, 1, device="cuda", generator=g) * w[y].float()).to(dtype)
    return h, w, y


def logits64(h, w):
    return h.double() @ w.double().t()


def logit_bound(h, w):
    """Per position: how far an fp32 sum of the products can be from the logit, at most."""
    k = h.shape[1]
    return (2 * k + 8) * E24 * (h.double().abs() @ w.double().abs().t()).amax(dim=1)


def check_forward(ext, h, w, y, ignore=IGNORE):
    loss, lse = ext.lm_head_cross_entropy(h, w, y, ignore)
    z = logits64(h, w)
    ref = torch.logsumexp(z, dim=1)
    vocab = w.shape[0]
    # the logits' error, the sum's (at most vocab additions, exponentials good to 2 steps, arguments to |z| steps)
    span = (z.amax(dim=1) - z.amin(dim=1)).abs() + ref.abs()
    tol = logit_bound(h, w) + (vocab + 64 + 4 * span) * E24
    assert loss.dtype == lse.dtype == torch.float32
    assert bool(((lse.double() - ref).abs() <= tol).all()), float(((lse.double() - ref).abs() - tol).max())
    counts = y != ignore
    at = torch.where(counts, y, 0).long()
    want = torch.where(counts, ref - z.gather(1, at[:, None]).squeeze(1), 0.0)
    assert bool(((loss.double() - want).abs() <= 2 * tol).all()), float(((loss.double() - want).abs() - 2 * tol).max())
    return loss, lse


def check_backward(ext, h, w, y, fwd, g, ignore=IGNORE, need_hidden=True, need_weight=True):
    gh, gw = ext.lm_head_cross_entropy_backward(g, h, w, y, *fwd, ignore, need_hidden, need_weight)
    assert (gh is not None) == need_hidden and (gw is not None) == need_weight
    dt = h.dtype
    u = U[dt]
    counts = (y != ignore).double()
    z = logits64(h, w)
    d = torch.softmax(z, dim=1)
    at = torch.where(y != ignore, y, 0).long()
    d[torch.arange(len(y), device=d.device), at] -= 1.0
    p = torch.softmax(z, dim=1)
    # an entry of p - [v = target]: the exponential's relative error, then one rounding to the 16-bit type
    span = (z.amax(dim=1) - z.amin(dim=1)).abs() + z.abs().amax(dim=1)
    rel = 2 * logit_bound(h, w) + (w.shape[0] + 128 + 8 * span) * E24
    # (fp16 holds it times 2^15)
    low = TINY[dt] * (2.0 ** -15 if dt == torch.float16 else 1.0)
    ed = u * d.abs() + rel[:, None] * p * (1 + u) + low
    hd = torch.where(counts[:, None] > 0, h.double(), 0.0)
    gd = (g.double() * counts)
    if need_hidden:
        want = gd[:, None] * (d @ w.double())
        acc = (2 * w.shape[0] + 64) * E24
        tol = gd.abs()[:, None] * ((ed + acc * d.abs()) @ w.double().abs())
        tol = tol + u * (want.abs() + tol) + TINY[dt]
        assert gh.dtype == dt and gh.shape == h.shape
        assert bool(((gh.double() - want).abs() <= tol).all()), float(((gh.double() - want).abs() - tol).max())
        assert bool((gh[y == ignore] == 0).all())
    if need_weight:
        want = (gd[:, None] * d).t().contiguous() @ hd
        acc = (2 * h.shape[0] + 64) * E24
        # a hidden row times g / max g is rounded to the 16-bit type too
        top = gd.abs().max()
        mag = (gd.abs()[:, None] * (ed + (acc + 2 * u) * d.abs())).t().contiguous() @ hd.abs()
        tol = mag + top * TINY[dt] * d.abs().sum(dim=0)[:, None]
        tol = tol + u * (want.abs() + tol) + TINY[dt]
        assert gw.dtype == dt and gw.shape == w.shape
        assert bool(((gw.double() - want).abs() <= tol).all()), float(((gw.double() - want).abs() - tol).max())
    return gh, gw


DTYPES = [torch.float16, torch.bfloat16]
SIZES = [  # tokens, vocabulary, width: single ones, one less and one more than tiles and K steps, odd ones
    (1, 1, 8), (1, 5000, 1024), (2, 127, 64), (31, 129, 72), (33, 1000, 584), (63, 257, 8), (64, 128, 128), (65, 1021, 136),
    (127, 2048, 56), (128, 4001, 1024), (129, 255, 248), (200, 30011, 64), (255, 513, 512), (257, 777, 1032), (700, 3001, 320),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,vocab,width", SIZES)
def test_cross_entropy_and_gradients(ext, tokens, vocab, width, dtype):
    h, w, y = make(tokens, vocab, width, dtype, seed=tokens)
    fwd = check_forward(ext, h, w, y)
    g = torch.rand(tokens, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) + 0.5
    check_backward(ext, h, w, y, fwd, g)


@pytest.mark.parametrize("dtype", DTYPES)
def test_full_head(ext, dtype):
    h, w, y = make(130, 151936, 1024, dtype, seed=5)
    fwd = check_forward(ext, h, w, y)
    check_backward(ext, h, w, y, fwd, torch.full((130,), 8.0, device="cuda"))


def test_several_pieces_of_the_vocabulary(ext):
    """More positions than let the whole vocabulary's gradient be kept at once."""
    h, w, y = make(4100, 40009, 64, torch.bfloat16, seed=6)
    fwd = check_forward(ext, h, w, y)
    check_backward(ext, h, w, y, fwd, torch.full((4100,), 0.25, device="cuda"))


def test_same_bits_every_time(ext):
    h, w, y = make(300, 5003, 256, torch.bfloat16, seed=7)
    g = torch.rand(300, device="cuda", generator=torch.Generator(device="cuda").manual_seed(8))
    fwd = ext.lm_head_cross_entropy(h, w, y)
    first = (*fwd, *ext.lm_head_cross_entropy_backward(g, h, w, y, *fwd))
    for _ in range(3):
        fwd = ext.lm_head_cross_entropy(h, w, y)
        again = (*fwd, *ext.lm_head_cross_entropy_backward(g, h, w, y, *fwd))
        assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("tokens", [1, 70, 140, 300])
def test_rows_further_apart_than_long(ext, tokens):
    """Rows of a wider array; the numbers between them are NaN and must not be read into anything."""
    h, w, y = make(tokens, 1001, 200, torch.float16, seed=9, pad=24)
    for t in (h, w):
        base = t._base if t._base is not None else t
        base[:, 200:] = float("nan")
    assert h.stride(0) == 224 and not h.is_contiguous() or tokens == 1
    fwd = check_forward(ext, h, w, y)
    check_backward(ext, h, w, y, fwd, torch.ones(tokens, device="cuda"))


@pytest.mark.parametrize("dtype", DTYPES)
def test_positions_that_do_not_count(ext, dtype):
    """Their hidden rows may hold NaN; they get zero rows and leave grad_weight alone. int32 targets."""
    h, w, y = make(200, 3001, 128, dtype, seed=10)
    y[::3] = IGNORE
    y[64:130] = IGNORE
    clean = check_forward(ext, h, w, y)
    want = check_backward(ext, h, w, y, clean, torch.ones(200, device="cuda"))
    bad = h.clone()
    bad[y == IGNORE] = float("nan")
    fwd = ext.lm_head_cross_entropy(bad, w, y.int())
    assert torch.equal(fwd[0], clean[0]) and bool((fwd[0][y == IGNORE] == 0).all())
    got = ext.lm_head_cross_entropy_backward(torch.ones(200, device="cuda"), bad, w, y.int(), *fwd)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_ignore_index_that_is_a_row_of_the_head(ext):
    h, w, y = make(90, 50, 64, torch.float16, seed=11)
    assert bool((y == 7).any())
    fwd = check_forward(ext, h, w, y, ignore=7)
    check_backward(ext, h, w, y, fwd, torch.ones(90, device="cuda"), ignore=7)


def test_no_position_counts(ext):
    import Qwen06B_architecture as qa

    h, w, _ = make(70, 300, 64, torch.float16, seed=12)
    y = torch.full((70,), IGNORE, device="cuda")
    loss, lse = ext.lm_head_cross_entropy(h, w, y)
    assert bool((loss == 0).all()) and bool(torch.isfinite(lse).all())
    h.requires_grad_()
    w.requires_grad_()
    for reduction in ("mean", "sum"):
        out = qa.lm_head_loss(h, w, y, reduction=reduction)
        value = float(out.detach())
        assert math.isnan(value) if reduction == "mean" else value == 0
        grads = torch.autograd.grad(out, [h, w])
        assert all(bool((x == 0).all()) for x in grads)


def test_no_positions(ext):
    import Qwen06B_architecture as qa

    h = torch.empty(0, 64, device="cuda", dtype=torch.float16, requires_grad=True)
    w = torch.randn(100, 64, device="cuda").half().requires_grad_()
    y = torch.empty(0, device="cuda", dtype=torch.int64)
    loss, lse = ext.lm_head_cross_entropy(h.detach(), w.detach(), y)
    assert loss.shape == lse.shape == (0,)
    out = qa.lm_head_loss(h, w, y, reduction="sum")
    assert float(out.detach()) == 0
    gh, gw = torch.autograd.grad(out, [h, w])
    assert gh.shape == h.shape and bool((gw == 0).all())
    assert math.isnan(float(qa.lm_head_loss(h, w, y).detach()))


def test_target_outside_the_head(ext):
    """Neither a row nor ignore_index: NaN loss, for that position alone."""
    h, w, y = make(40, 300, 64, torch.float16, seed=13)
    y[3], y[17] = 300, -1
    loss, lse = ext.lm_head_cross_entropy(h, w, y)
    nan = torch.isnan(loss).nonzero().flatten().tolist()
    assert nan == [3, 17] and bool(torch.isfinite(lse).all())
    gh, _ = ext.lm_head_cross_entropy_backward(torch.ones(40, device="cuda"), h, w, y, loss, lse, need_weight=False)
    assert torch.isnan(gh).any(dim=1).nonzero().flatten().tolist() == [3, 17]


def test_logits_of_the_lowest_value_and_infinite_ones(ext):
    """-inf logits have probability 0; a position whose logits are all -inf, or one +inf, has a NaN loss."""
    vocab = 700
    w = torch.zeros(vocab, 64, device="cuda", dtype=torch.float16)
    w[:, 0] = 1.0
    w[5:400, 1] = float("-inf")
    h = torch.zeros(3, 64, device="cuda", dtype=torch.float16)
    h[:, 0] = 2.0
    h[1:, 1] = 1.0
    y = torch.tensor([1, 2, 6], device="cuda")
    # position 0 multiplies the -inf entries by 0: NaN, as the definition has it
    loss, lse = ext.lm_head_cross_entropy(h, w, y)
    assert math.isnan(float(loss[0]))
    assert abs(float(loss[1]) - math.log(305.0)) < 1e-5 and abs(float(lse[1]) - 2 - math.log(305.0)) < 1e-5
    assert float(loss[2]) == math.inf
    w[:, 1] = float("-inf")
    loss, _ = ext.lm_head_cross_entropy(h[1:], w, y[1:])
    assert bool(torch.isnan(loss).all())
    w[:, 1] = 0
    w[9, 1] = float("inf")
    loss, _ = ext.lm_head_cross_entropy(h[1:], w, torch.tensor([9, 3], device="cuda"))
    assert bool(torch.isnan(loss).all())


def test_loss_of_a_target_that_is_nearly_certain(ext):
    """log1p(others / target), not the difference of two equal numbers: relative accuracy down to 1e-30."""
    vocab = 1000
    w = torch.zeros(vocab, 64, device="cuda", dtype=torch.float16)
    w[123, 0] = 1.0
    h = torch.zeros(5, 64, device="cuda", dtype=torch.float16)
    h[:, 0] = torch.tensor([0.5, 8.0, 16.0, 40.0, 70.0], device="cuda").half()
    y = torch.full((5,), 123, device="cuda")
    loss, lse = ext.lm_head_cross_entropy(h, w, y)
    want = torch.log1p((vocab - 1) * torch.exp(-h[:, 0].double()))
    # the exponential's argument is rounded (to |logit| steps), then a few operations
    tol = (8 + 4 * h[:, 0].double()) * E24 * want
    assert bool(((loss.double() - want).abs() <= tol).all())
    gh, _ = ext.lm_head_cross_entropy_backward(torch.full((5,), 65536.0, device="cuda"), h, w, y, loss, lse,
                                               need_weight=False)
    d = -65536.0 * (1 - torch.exp(-want))  # the target's row is the only one with a nonzero entry
    tol = (2 * U[torch.float16] + 64 * E24) * d.abs() + TINY[torch.float16]
    assert bool(((gh[:, 0].double() - d).abs() <= tol).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,vocab,width", [(1, 5003, 1024), (2, 1001, 512), (3, 151936, 1024), (7, 300, 264), (65, 4001, 512),
                                                (256, 9001, 264), (700, 5003, 512)])
def test_gradients_of_few_positions_have_one_rounding(ext, tokens, vocab, width, dtype):
    """What G's rounding to 16 bits does to the targets' entries, the largest by far, is taken up again. With x the gradient
    before its own rounding and e = x - want, the rounding takes x to the nearest number, so |got - x| <= |round(want) - x|
    and |got - want| <= |round(want) - want| + 2 |e|. In norm, e is the other entries' roundings: each is off by at most
    U of itself, in both directions alike and independently, so the squares add up, sum (U d w)^2 (a third of it on average).
    The fp32 parts: logits up to 16, off by 2^-20 at most, move the entries by as much relative to them, and the sums add
    some 2^-22; 2^-13 / 4, the least that one rounding leaves in norm, is 2^-15, so that 2 |e| grows by 0.08 of it at most."""
    h, w, y = make(tokens, vocab, width, dtype, seed=70 + tokens, lean=4.0)
    if tokens > 5:
        y[4] = y[2]  # two positions with one target
    fwd = ext.lm_head_cross_entropy(h, w, y)
    scale = 1024.0  # (in fp16 small numbers would lose more than their rounding's half step)
    gh, gw = ext.lm_head_cross_entropy_backward(torch.full((tokens,), scale, device="cuda"), h, w, y, *fwd)
    d = torch.softmax(logits64(h, w), dim=1)
    d[torch.arange(tokens), y] -= 1.0
    other = d.clone()
    other[torch.arange(tokens), y] = 0.0
    for got, want, entries, rows in ((gh, scale * d @ w.double(), other, w),  # (past 256 positions grad_weight has them all)
                                     (gw, scale * d.t().contiguous() @ h.double(), (other if tokens <= 256 else d).t().contiguous(), h)):
        once = float((want.to(dtype).double() - want).norm())
        e = U[dtype] * scale * float(((entries ** 2) @ (rows.double() ** 2)).sum().sqrt())
        assert float((got.double() - want).norm()) <= 1.08 * once + 2 * e


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_of_an_impossible_target(ext, dtype):
    """A target whose row holds the lowest infinity: its loss is infinite, its entry -1 exactly, the gradient by the formula."""
    h, w, y = make(1, 300, 264, dtype, seed=5)
    h[0, 40] = 2.0
    w[y[0], 40] = -math.inf
    loss, lse = ext.lm_head_cross_entropy(h, w, y)
    gh, gw = ext.lm_head_cross_entropy_backward(torch.ones(1, device="cuda"), h, w, y, loss, lse)
    d = torch.softmax(logits64(h, w), dim=1)
    assert float(loss[0]) == math.inf and float(d[0, y[0]]) == 0.0
    assert float(gh[0, 40]) == math.inf  # -1 times the row's -inf
    d[0, y[0]] = -1.0
    want = d @ w.double()
    keep = torch.arange(264, device="cuda") != 40
    # each other entry is off by its rounding and by the sums' (2 n + 8) 2^-24, the result by a rounding (fp16: or 2^-25)
    tol = (U[dtype] + 2.0 ** -14) * (d.abs() @ w.double().abs()) + U[dtype] * want.abs() + 2.0 ** -25
    assert bool(((gh.double() - want).abs() <= tol)[0, keep].all())
    assert torch.equal(gw[y[0]], -h[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_lm_head_loss(ext, dtype, reduction):
    import Qwen06B_architecture as qa

    h, w, y = make(150, 2003, 192, dtype, seed=14)
    y[5:40] = IGNORE
    up = 64.0
    hx, wx = h.detach().requires_grad_(), w.detach().requires_grad_()
    out = qa.lm_head_loss(hx, wx, y, reduction=reduction)
    weights = torch.ones(150, device="cuda") if reduction != "none" else torch.linspace(-1, 2, 150, device="cuda")
    scalar = (out * weights).sum() if reduction == "none" else out
    gh, gw = torch.autograd.grad(scalar * up, [hx, wx])
    loss, lse = ext.lm_head_cross_entropy(h, w, y)
    g = weights * up / (115 if reduction == "mean" else 1)
    if reduction == "none":
        assert torch.equal(out, loss)
    else:
        want = float(loss.double().sum()) / (115 if reduction == "mean" else 1)
        assert abs(float(out.detach()) - want) <= 160 * E24 * abs(want)
    wh, ww = check_backward(ext, h, w, y, (loss, lse), g)
    # the same gradients (for the mean but for the rounding of its division)
    assert bool(((gh.double() - wh.double()).abs() <= 4 * U[dt_of(gh)] * wh.double().abs() + TINY[dt_of(gh)]).all())
    assert bool(((gw.double() - ww.double()).abs() <= 4 * U[dt_of(gw)] * ww.double().abs() + TINY[dt_of(gw)]).all())
    # one leaf at a time
    only_h = torch.autograd.grad((qa.lm_head_loss(hx, w, y, reduction=reduction) * weights * up).sum()
                                 if reduction == "none" else qa.lm_head_loss(hx, w, y, reduction=reduction) * up, [hx])
    assert torch.equal(only_h[0], gh)
    only_w = torch.autograd.grad((qa.lm_head_loss(h, wx, y, reduction=reduction) * weights * up).sum()
                                 if reduction == "none" else qa.lm_head_loss(h, wx, y, reduction=reduction) * up, [wx])
    assert torch.equal(only_w[0], gw)


def test_lm_head_loss_changed_in_place_and_its_second_derivative(ext):
    import Qwen06B_architecture as qa

    h, w, y = make(50, 300, 64, torch.float16, seed=18)
    h.requires_grad_()
    for reduction in ("mean", "sum"):
        want = torch.autograd.grad(qa.lm_head_loss(h, w, y, reduction=reduction) / 4, [h])[0]
        loss = qa.lm_head_loss(h, w, y, reduction=reduction)
        value = float(loss.detach())
        loss /= 4
        assert float(loss.detach()) == value / 4
        assert torch.equal(torch.autograd.grad(loss, [h])[0], want)
    # every position's losses are what the gradients are made of: changed in place, they are missed
    loss = qa.lm_head_loss(h, w, y, reduction="none")
    loss *= 2
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(loss.sum(), [h])
    g, = torch.autograd.grad(qa.lm_head_loss(h, w, y), [h], create_graph=True)
    with pytest.raises(RuntimeError):  # (torch's own: h is not in what is left of the graph)
        torch.autograd.grad(g.float().sum(), [h], retain_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        (g.float().sum() + h.float().sum()).backward()
    # nothing to differentiate, and no graph wanted
    assert not qa.lm_head_loss(h.detach(), w, y).requires_grad
    with torch.no_grad():
        assert not qa.lm_head_loss(h, w, y).requires_grad
    # accumulated over two calls, as a training loop does
    h.grad = None
    for _ in range(2):
        (qa.lm_head_loss(h, w, y) * 64).backward()
    one = torch.autograd.grad(qa.lm_head_loss(h, w, y) * 64, [h])[0]
    assert torch.equal(h.grad, one + one)


def dt_of(t):
    return t.dtype


def test_gradient_against_differences(ext):
    """Central differences of the loss along a direction: their own error is bounded by the third derivative of
    log-sum-exp, at most R^3 / (6 sqrt 3) for logits that move by a range R."""
    h, w, y = make(60, 1500, 128, torch.float16, seed=15)
    h = (h.float() * 64).round().div(64).half()  # so that h +- step is exact
    step = (torch.randint(0, 2, h.shape, device="cuda").float() * 2 - 1).div(64)
    up, down = (h.float() + step).half(), (h.float() - step).half()
    assert torch.equal(up.float() - h.float(), step) and torch.equal(h.float() - down.float(), step)
    loss, lse = ext.lm_head_cross_entropy(h, w, y)
    diff = (ext.lm_head_cross_entropy(up, w, y)[0].double() - ext.lm_head_cross_entropy(down, w, y)[0].double()) / 2
    gh, _ = ext.lm_head_cross_entropy_backward(torch.full((60,), 256.0, device="cuda"), h, w, y, loss, lse, need_weight=False)
    got = (gh.double() / 256 * step.double()).sum(dim=1)
    move = step.double() @ w.double().t()
    r = move.amax(dim=1) - move.amin(dim=1)
    e_grad = ((2 * U[torch.float16]) * gh.double().abs() / 256 * step.abs()).sum(dim=1)
    # ... and what G's own rounding does to a row: u sum |G| |w|, with sum |G| <= 2
    e_grad = e_grad + U[torch.float16] * 2 * (w.double().abs().amax(dim=0) * step.abs().double()).sum(dim=1)
    tol = r ** 3 / (36 * math.sqrt(3)) + 2 * logit_bound(h, w) + 64 * E24 * lse.double().abs() + e_grad
    assert bool(((diff - got).abs() <= tol).all())
    assert float(diff.abs().max()) > 20 * float(tol.max())  # the comparison says something


# ---- 8-bit integers


def quantize64(x):
    x = x.double()
    top = x.abs().amax(dim=1)
    q = torch.round(127 * x / torch.where(top > 0, top, torch.ones_like(top))[:, None])
    return q, top / 127


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width,pad", [(1, 16, 0), (3, 512, 0), (5, 528, 0), (127, 2048, 0), (1000, 1024, 0),
                                            (33, 1040, 24), (4, 12288, 0), (2, 65536, 0)])
def test_quantize_rows(ext, rows, width, pad, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, width + pad, device="cuda", generator=g).to(dtype)[:, :width]
    x *= torch.logspace(-4, 3, rows, device="cuda")[:, None].to(dtype)
    q, scale = ext.quantize_rows(x)
    want, unit = quantize64(x)
    assert q.dtype == torch.int8 and torch.equal(q.double(), want)
    assert bool(((scale.double() - unit).abs() <= E24 * unit).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_rows_ties_and_extremes(ext, dtype):
    x = torch.zeros(8, 64, device="cuda")
    x[0, :40] = torch.arange(-20, 20, device="cuda") + 0.5  # ties, with a scale of 1
    x[0, 63] = 127
    x[1] = 0.0  # zeros
    x[2, 5] = float("inf")
    x[3, 60] = float("nan")
    x[4, 7] = float("-inf")
    big = torch.finfo(dtype).max
    x[5, :3] = torch.tensor([1.0, -0.5, 0.25], device="cuda") * big
    tiny = float(TINY[dtype])
    x[6, :4] = torch.tensor([4, -2, 1, 3], device="cuda") * tiny  # subnormal numbers
    x[7, :2] = torch.tensor([1e-3, 5.0], device="cuda")
    x = x.to(dtype)
    q, scale = ext.quantize_rows(x)
    ok = [0, 1, 5, 6, 7]
    want, unit = quantize64(x[ok])
    assert torch.equal(q[ok].double(), want)
    # (a scale in fp32's own subnormal range is exact to half its step)
    assert bool(((scale[ok].double() - unit).abs() <= E24 * unit + 2.0 ** -150).all())
    assert float(scale[1]) == 0
    assert bool(torch.isnan(scale[[2, 3, 4]]).all()) and bool((q[[2, 3, 4]] == 0).all())


@pytest.mark.parametrize("out", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,rows,width", [
    (1, 1, 16), (1, 5000, 1024), (2, 63, 48), (15, 4096, 1024), (31, 65, 128), (64, 64, 64), (65, 129, 144), (127, 1000, 2048),
    (128, 256, 1040), (129, 4097, 256), (257, 513, 1024), (700, 3001, 112), (1000, 9000, 80), (40, 30, 65536),
])
def test_matmul_i8(ext, tokens, rows, width, out):
    g = torch.Generator(device="cuda").manual_seed(tokens)
    a = torch.randint(-128, 128, (tokens, width), device="cuda", dtype=torch.int8, generator=g)
    b = torch.randint(-128, 128, (rows, width), device="cuda", dtype=torch.int8, generator=g)
    if width == 65536:
        a[0], b[0] = -128, -128  # the largest sum, 2^30
    sa = torch.rand(tokens, device="cuda", generator=g) / width ** 0.5 / 32
    sb = torch.rand(rows, device="cuda", generator=g) / 32
    got = ext.matmul_i8(a, sa, b, sb, out)
    want = (a.double() @ b.double().t()) * sa.double()[:, None] * sb.double()
    u = U.get(out, 0.0)
    tiny = TINY.get(out, 2.0 ** -149)
    # the sum to fp32, two products, then the output's own rounding
    tol = (3 * E24 * 1.001 + u) * want.abs() + tiny
    assert got.dtype == out and got.shape == (tokens, rows)
    assert bool(((got.double() - want).abs() <= tol).all())


def test_matmul_i8_nothing_to_do(ext):
    e = torch.empty(0, 64, device="cuda", dtype=torch.int8)
    b = torch.ones(5, 64, device="cuda", dtype=torch.int8)
    s0, s5 = torch.empty(0, device="cuda"), torch.ones(5, device="cuda")
    assert ext.matmul_i8(e, s0, b, s5).shape == (0, 5)
    assert ext.matmul_i8(b, s5, e, s0).shape == (5, 0)
    q, s = ext.quantize_rows(torch.empty(0, 64, device="cuda", dtype=torch.float16))
    assert q.shape == (0, 64) and s.shape == (0,)


def test_matmul_i8_scales_of_nan(ext):
    """A row that held an infinity makes its products NaN, and no others."""
    x = torch.randn(70, 128, device="cuda").half()
    x[9, 3] = float("inf")
    w = torch.randn(200, 128, device="cuda").half()
    w[150, 0] = float("nan")
    out = ext.matmul_i8(*ext.quantize_rows(x), *ext.quantize_rows(w), torch.float32)
    bad = torch.isnan(out)
    want = torch.zeros_like(bad)
    want[9] = True
    want[:, 150] = True
    assert torch.equal(bad, want)


# ---- together, on streams and in graphs


def test_a_step_of_all_of_them_captured_and_replayed(ext):
    """Loss, gradients, and 8-bit logits of the same rows, on a stream and in a graph whose inputs change."""
    h, w, y = make(300, 4001, 256, torch.bfloat16, seed=16)
    g = torch.full((300,), 0.5, device="cuda")

    def step():
        fwd = ext.lm_head_cross_entropy(h, w, y)
        grads = ext.lm_head_cross_entropy_backward(g, h, w, y, *fwd)
        out = ext.matmul_i8(*ext.quantize_rows(h), *ext.quantize_rows(w), torch.bfloat16)
        return (*fwd, *grads, out)

    eager = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, on_side))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    other = torch.cuda.CUDAGraph()  # a second graph, with workspaces of its own
    with torch.cuda.graph(other):
        captured2 = step()
    for k in range(4):
        h.copy_(make(300, 4001, 256, torch.bfloat16, seed=20 + k)[0])
        graph.replay()
        other.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, captured)), k
        assert all(torch.equal(a, b) for a, b in zip(eager, captured2)), k


def test_loss_and_gradients_captured_through_autograd(ext):
    """A training step in a graph, its gradients taken with torch.autograd.grad; inputs change between replays."""
    import Qwen06B_architecture as qa

    h, w, y = make(200, 2003, 192, torch.float16, seed=17)
    y[::4] = IGNORE

    def step():
        hx, wx = h.detach().requires_grad_(), w.detach().requires_grad_()
        loss = qa.lm_head_loss(hx, wx, y)
        return (loss.detach(), *torch.autograd.grad(loss * 512.0, [hx, wx]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm up on the side, as torch asks for
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(3):
        new = make(200, 2003, 192, torch.float16, seed=50 + k)
        h.copy_(new[0])
        w.copy_(new[1])
        y[1::4] = new[2][1::4]
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, eager)), k


def test_two_threads(ext):
    """Calls from two threads, each on a stream of its own."""
    import threading

    data = [make(260, 3001, 128, torch.float16, seed=30 + k) for k in range(2)]
    want = []
    for h, w, y in data:
        fwd = ext.lm_head_cross_entropy(h, w, y)
        want.append((*fwd, *ext.lm_head_cross_entropy_backward(torch.ones(260, device="cuda"), h, w, y, *fwd)))
    torch.cuda.synchronize()
    wrong = []

    def run(k):
        try:
            stream = torch.cuda.Stream()
            h, w, y = data[k]
            with torch.cuda.stream(stream):
                one = torch.ones(260, device="cuda")
                for _ in range(20):
                    fwd = ext.lm_head_cross_entropy(h, w, y)
                    got = (*fwd, *ext.lm_head_cross_entropy_backward(one, h, w, y, *fwd))
                    stream.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[k])):
                        wrong.append(k)
        except Exception as e:  # noqa: BLE001
            wrong.append(repr(e))

    threads = [threading.Thread(target=run, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong


# ---- refusals


def test_refusals(ext):
    h, w, y = make(8, 32, 64, torch.float16)
    loss, lse = ext.lm_head_cross_entropy(h, w, y)
    one = torch.ones(8, device="cuda")
    bad = [
        (h.float(), w, y), (h, w.bfloat16(), y), (h.cpu(), w, y), (h, w.cpu(), y), (h, w, y.cpu()), (h, w, y.short()),
        (h, w, y[:7]), (h, w[:, :56], y), (h[:, :60], w[:, :60], y), (h, w[:0], y), (h.t(), w, y), (h[0], w, y),
        (h[:, 1:57], w[:, 1:57], y),  # rows that do not begin on 16 bytes
        (torch.empty(8, 68, device="cuda", dtype=torch.float16)[:, :64], w, y),  # rows 136 bytes apart
    ]
    for args in bad:
        with pytest.raises(RuntimeError):
            ext.lm_head_cross_entropy(*args)
        with pytest.raises(RuntimeError):
            ext.lm_head_cross_entropy_backward(one, *args, loss, lse)
    for args in ((one[:7], h, w, y, loss, lse), (one.half(), h, w, y, loss, lse), (one, h, w, y, loss[:7], lse),
                 (one, h, w, y, loss, lse.double()), (one.cpu(), h, w, y, loss, lse)):
        with pytest.raises(RuntimeError):
            ext.lm_head_cross_entropy_backward(*args)
    with pytest.raises(RuntimeError):
        ext.lm_head_cross_entropy_backward(one, h, w, y, loss, lse, divisor=one)
    for x in (h.float(), h.cpu(), h[:, :24], h[0], h.t()):
        with pytest.raises(RuntimeError):
            ext.quantize_rows(x)
    q, s = ext.quantize_rows(h)
    wq, ws = ext.quantize_rows(w)
    for args in ((q.int(), s, wq, ws), (q, s[:7], wq, ws), (q, s.half(), wq, ws), (q[:, :48], s, wq[:, :48], ws),
                 (q, s, wq[:, :48].contiguous(), ws), (q.cpu(), s, wq, ws), (q, s.cpu(), wq, ws),
                 (q[:, :24].contiguous(), s, wq[:, :24].contiguous(), ws)):
        with pytest.raises(RuntimeError):
            ext.matmul_i8(*args)
    with pytest.raises(RuntimeError):
        ext.matmul_i8(q, s, wq, ws, torch.float64)
    import Qwen06B_architecture as qa

    with pytest.raises(ValueError):
        qa.lm_head_loss(h, w, y, reduction="max")


# ---- the engine's own paths


@pytest.fixture(scope="module")
def decoder():
    import Qwen06B_architecture as qa
    import qwen_weights as qw

    shape = qw.QwenShape(layers=2)
    return qa.Decoder(weights=qw.device_weights(qw.host_weights(seed=0, shape=shape, norms="random")))


@pytest.mark.parametrize("n", [2, 17, 130, 600, 1100])
def test_score_against_the_decode_kernels_logits(ext, decoder, n):
    """The prompt's log-probabilities from one prefill, and from the logits that the decode kernel gives id by
    id (teacher forced). The two paths round activations to fp16 at different places: the logits agree to 5e-2, as
    in the parity tests, so a log-probability to twice that."""
    import qwen_weights as qw

    ids = qw.synthetic_prompt(n, seed=n)
    got = decoder.score(ids)
    assert got.shape == (n - 1,) and decoder.position == n - 1
    steps = min(n - 1, 64)
    decoder.reset()
    forced = torch.tensor(ids[:steps], dtype=torch.int32, device="cuda")
    logits = torch.empty(steps, 151936, device="cuda")
    ext.generate_ex(ids[0], steps, forced, decoder._embed_weight, decoder._layer_weights_packed, decoder._final_norm_weight,
                    decoder._lm_head_weight, decoder._cos_table, decoder._sin_table, decoder._k_cache, decoder._v_cache,
                    decoder._hidden, decoder._norm_out, logits, None, decoder._num_layers, 0, 2048, decoder._attn_scale)
    torch.cuda.synchronize()
    assert ext.last_error() == 0
    want = torch.log_softmax(logits.double(), dim=1)[torch.arange(steps), torch.tensor(ids[1:steps + 1], device="cuda")]
    assert float((got[:steps].double() - want).abs().max()) < 0.1


def test_hidden_states_and_8_bit_logits(ext, decoder):
    import qwen_weights as qw

    ids = qw.synthetic_prompt(300, seed=3)
    decoder.reset()
    whole = decoder.hidden_states(ids)
    assert whole.shape == (300, 1024) and whole.dtype == torch.float16 and decoder.position == 300
    decoder.reset()
    pieces = torch.cat([decoder.hidden_states(ids[:77]), decoder.hidden_states(ids[77:])])
    assert torch.equal(whole, pieces)
    head8 = decoder.quantize_head()
    decoder.reset()
    got = decoder.logits(ids, head8)
    q, s = quantize64(whole)
    # the definition, from the rows' and the head's own roundings. The sums are whole numbers below 2^53, so exact here;
    # the engine rounds the sum, the row's scale, the product of the scales and the result to fp32: (1 + E24)^4
    want = (q @ head8[0].double().t().contiguous()) * s[:, None] * head8[1].double()
    assert got.shape == (300, 151936) and got.dtype == torch.float32
    assert bool(((got.double() - want).abs() <= 4.001 * E24 * want.abs()).all())
    # and against the 16-bit head: half a step of each factor's 8-bit grid, times the other's size
    exact = whole.double() @ decoder._lm_head_weight.double().t()
    w = decoder._lm_head_weight.double()
    bound = 0.5 * s[:, None] * w.abs().sum(dim=1) + 0.5 * head8[1].double() * (q.abs() * s[:, None]).sum(dim=1)[:, None]
    assert bool(((got.double() - exact).abs() <= 1.001 * bound + 1e-6).all())


def test_hidden_states_captured_and_replayed(ext, decoder):
    """The prefill and the norm that reads its workspace, as nodes of a graph between calls of other lengths."""
    import qwen_weights as qw

    d = decoder

    def call(t, n):
        return ext.prefill_hidden(t, d._embed_weight, d._layer_weights_packed, d._final_norm_weight, d._cos_table, d._sin_table,
                                  d._k_cache, d._v_cache, d._hidden, d._num_layers, 0, 2048, d._attn_scale)

    texts = [torch.tensor(qw.synthetic_prompt(150, seed=60 + k), dtype=torch.int32, device="cuda") for k in range(3)]
    want = [call(t, 150).clone() for t in texts]
    ids = texts[0].clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        rows = call(ids, 150)
    for k in (1, 2, 0, 1):
        ids.copy_(texts[k])
        graph.replay()
        other = call(texts[(k + 1) % 3], 150)  # right after it, on the same workspace
        torch.cuda.synchronize()
        assert torch.equal(rows, want[k]) and torch.equal(other, want[(k + 1) % 3]), k
    assert ext.last_error() == 0


def test_two_streams_of_hidden_states(ext, decoder):
    """The second call's prefill waits for the first one's norm, which reads the shared workspace."""
    import qwen_weights as qw

    ids = [qw.synthetic_prompt(n, seed=n) for n in (900, 880)]
    caches = [(torch.zeros_like(decoder._k_cache), torch.zeros_like(decoder._v_cache)) for _ in ids]
    hidden = [torch.empty_like(decoder._hidden) for _ in ids]
    d = decoder

    def call(k):
        t = torch.tensor(ids[k], dtype=torch.int32, device="cuda")
        return ext.prefill_hidden(t, d._embed_weight, d._layer_weights_packed, d._final_norm_weight, d._cos_table, d._sin_table,
                                  *caches[k], hidden[k], d._num_layers, 0, 2048, d._attn_scale)

    want = [call(0), call(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        got = []
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(call(k))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_decoder_refusals(decoder):
    for call in (lambda: decoder.score([5]), lambda: decoder.score([5, 151936]), lambda: decoder.score([-1, 5]),
                 lambda: decoder.hidden_states([])):
        with pytest.raises(ValueError):
            call()
    decoder.reset()
    with pytest.raises(RuntimeError):
        decoder.hidden_states([1] * 2049)


def test_training_a_head_on_the_engines_hidden_rows(ext, decoder):
    """Hidden rows of two texts, a loss with padding, gradients for the head and for what stands before it."""
    import Qwen06B_architecture as qa
    import qwen_weights as qw

    rows, targets = [], []
    for k, n in enumerate((90, 33)):
        ids = qw.synthetic_prompt(n, seed=40 + k)
        decoder.reset()
        rows.append(decoder.hidden_states(ids))
        targets.append(torch.tensor(ids[1:] + [IGNORE], device="cuda"))
    h, y = torch.cat(rows).requires_grad_(), torch.cat(targets)
    w = decoder._lm_head_weight.detach().clone().requires_grad_()
    loss = qa.lm_head_loss(h, w, y)
    gh, gw = torch.autograd.grad(loss * 1024.0, [h, w])
    fwd = ext.lm_head_cross_entropy(h.detach(), w.detach(), y)
    want = check_backward(ext, h.detach(), w.detach(), y, fwd, torch.full((123,), 1024.0 / 121, device="cuda"))
    for a, b in zip((gh, gw), want):
        assert bool(((a.double() - b.double()).abs() <= 4 * U[torch.float16] * b.double().abs() + TINY[torch.float16]).all())
