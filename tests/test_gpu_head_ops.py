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
