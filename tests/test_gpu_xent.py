"""Softmax cross entropy of a classifier and its gradient on the GPU against a plain implementation in 64 bits, within
bounds that follow from the arithmetic (xent_ref)."""
import numpy as np
import pytest

import xent_ref
from ulmblas_amd import blas

pytestmark = pytest.mark.gpu

IGNORE = -100


def window(A, prec, pad, off, fill=float("nan")):
    """A [rows, cols] matrix as a device window with row stride cols + pad, `off` elements into its memory; the
    memory around it holds `fill`.  Returns (tensor of the window, its 64-bit values, stride)."""
    import torch
    dt = {"s": torch.float32, "b": torch.bfloat16}[prec]
    rows, cols = A.shape
    ld = cols + pad
    flat = torch.full((off + rows * ld + 64,), fill, dtype=dt, device="cuda")
    view = flat[off:off + rows * ld].view(rows, ld)[:, :cols]
    view.copy_(torch.from_numpy(A).to(dt))
    return view, view.double().cpu().numpy(), ld


class Problem:
    def __init__(self, prec, hidden, tokens, vocab, pad=0, off=0, alpha=1.0, masked=0.0, seed=0, spread=1.5):
        import torch
        rng = np.random.default_rng(seed)
        W = rng.standard_normal((vocab, hidden)) * (2.0 / np.sqrt(hidden))
        label = rng.integers(0, vocab, tokens)
        X = rng.standard_normal((tokens, hidden)) + spread * W[label]
        drop = rng.random(tokens) < masked
        label[drop] = np.resize(np.array([IGNORE, -1, vocab, 2 ** 31 - 1, -2 ** 31]), int(drop.sum()))
        X[drop] = np.resize(np.array([np.nan, np.inf, -np.inf, 1.0]), (int(drop.sum()), 1))
        self.prec, self.H, self.T, self.V, self.alpha = prec, hidden, tokens, vocab, alpha
        self.label = label
        self.W, self.w64, self.ldW = window(W, prec, pad, off)
        self.X, self.x64, self.ldX = window(X, prec, pad, off)
        self.dlabel = torch.from_numpy(label.astype(np.int32)).cuda()
        self.gloss = (rng.standard_normal(tokens) / max(tokens, 1)).astype(np.float32)
        self.glse = (rng.standard_normal(tokens) * 0.1 / max(tokens, 1)).astype(np.float32)
        self.rng = rng

    def work(self, size):
        """A workspace whose every word is NaN."""
        import torch
        return torch.full((size,), 0xff, dtype=torch.uint8, device="cuda")

    def forward(self, stream=None):
        import torch
        loss, lse = (torch.full((self.T + 3,), 7.5, device="cuda") for _ in range(2))
        work = self.work(blas.xent_worksize(self.prec, self.H, self.T, self.V))
        blas.gpu_xent(self.prec, self.H, self.T, self.V, self.alpha, self.W, self.ldW, self.X, self.ldX, self.dlabel,
                      IGNORE, loss, lse, work=work, stream=stream)
        torch.cuda.synchronize()
        assert (loss[self.T:] == 7.5).all() and (lse[self.T:] == 7.5).all()
        return loss[:self.T].double().cpu().numpy(), lse[:self.T].double().cpu().numpy()

    def check_forward(self):
        loss, lse = self.forward()
        x64 = np.where(xent_ref.valid(self.label, self.V, IGNORE)[:, None], self.x64, 0.0)
        wloss, wlse, blse, bloss = xent_ref.forward(self.w64, x64, self.label, self.alpha, IGNORE, self.prec)
        assert np.isfinite(loss).all() and np.isfinite(lse).all()
        assert (np.abs(lse - wlse) <= blse).all(), np.nanmax(np.abs(lse - wlse) / blse)
        assert (np.abs(loss - wloss) <= bloss).all(), np.nanmax(np.abs(loss - wloss) / bloss)
        return lse

    def check_backward(self, glse=True, beta=0.0, want=("W", "X"), pad_out=0, off_out=0):
        import torch
        x64 = np.where(xent_ref.valid(self.label, self.V, IGNORE)[:, None], self.x64, 0.0)
        lse = xent_ref.forward(self.w64, x64, self.label, self.alpha, IGNORE, self.prec)[1].astype(np.float32)
        gW0 = self.rng.standard_normal((self.V, self.H)) if beta else np.full((self.V, self.H), np.nan)
        gW, gW64, ldGW = window(gW0, self.prec, pad_out, off_out, 3.25)
        gX, _, ldGX = window(np.full((self.T, self.H), np.nan), self.prec, pad_out, off_out, 3.25)
        work = self.work(blas.xent_grad_worksize(self.prec, self.H, self.T, self.V))
        # rows without a target may hold anything here too
        has = xent_ref.valid(self.label, self.V, IGNORE)
        f = [torch.from_numpy(np.where(has, a, np.float32(np.nan))).cuda() for a in (lse, self.gloss, self.glse)]
        blas.gpu_xent_grad(self.prec, self.H, self.T, self.V, self.alpha, self.W, self.ldW, self.X, self.ldX, self.dlabel,
                           IGNORE, f[0], f[1], f[2] if glse else None, beta, gW if "W" in want else None, ldGW,
                           gX if "X" in want else None, ldGX, work=work)
        torch.cuda.synchronize()
        wW, wX, bW, bX = xent_ref.backward(self.w64, x64, self.label, self.alpha, IGNORE, lse.astype(np.float64),
                                           self.gloss.astype(np.float64),
                                           self.glse.astype(np.float64) if glse else None, self.prec, beta,
                                           gW64 if beta else None)
        for name, got, want64, bound in (("W", gW, wW, bW), ("X", gX, wX, bX)):
            g = got.double().cpu().numpy()
            if name not in want:
                assert np.isnan(g).all() or beta, name
                continue
            assert np.isfinite(g).all(), name
            d = np.abs(g - want64)
            assert (d <= bound).all(), (name, float((d / bound).max()))
            # the memory around the window is as it was
            flat = got.untyped_storage()
            whole = torch.empty(0, dtype=got.dtype, device="cuda").set_(flat)
            inside = torch.zeros_like(whole, dtype=torch.bool)
            torch.as_strided(inside, got.shape, got.stride(), got.storage_offset())[:] = True
            assert (whole[~inside] == 3.25).all(), name
        if "X" in want:
            assert (gX.double().cpu().numpy()[~has] == 0).all()
        return gW, gX


SIZES = [  # hidden, tokens, vocab
    (1, 1, 1), (8, 1, 2), (64, 1, 1000), (65, 7, 257), (96, 16, 300), (72, 17, 4097), (200, 33, 640), (1000, 130, 777),
    (512, 300, 5000), (40, 257, 511), (4097, 3, 130), (300, 8, 9000), (72, 9, 2049), (8200, 2, 300),
]


@pytest.mark.parametrize("prec", ["s", "b"])
@pytest.mark.parametrize("hidden,tokens,vocab", SIZES)
def test_sizes(prec, hidden, tokens, vocab):
    p = Problem(prec, hidden, tokens, vocab, seed=hidden + tokens)
    p.check_forward()
    p.check_backward()


@pytest.mark.parametrize("prec", ["s", "b"])
@pytest.mark.parametrize("hidden", [7, 511, 513, 4096, 4097, 8191])
@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 6, 8])
def test_few_tokens(prec, hidden, tokens):
    """One pass over W, for every number of tokens, one and two stretches of elements a thread."""
    p = Problem(prec, hidden, tokens, 67, pad=hidden % 3, off=hidden % 5, seed=hidden + tokens, masked=0.3)
    p.check_forward()
    p.check_backward(beta=0.5, pad_out=1)
    p.check_backward(glse=False, want=("X",))
    p.check_backward(want=("W",))


@pytest.mark.parametrize("prec", ["s", "b"])
def test_large_tiles(prec):
    """Sizes that take the 256 x 256 tile in every product."""
    p = Problem(prec, 128, 300, 26000, seed=5, masked=0.1)
    p.check_forward()
    p.check_backward()
    q = Problem(prec, 1800, 6500, 1900, seed=6, masked=0.5)
    q.check_forward()
    q.check_backward()


@pytest.mark.parametrize("prec", ["s", "b"])
@pytest.mark.parametrize("pad,off", [(1, 0), (0, 1), (8, 8), (3, 5)])
def test_strides_and_alignment(prec, pad, off):
    for hidden, tokens, vocab in ((128, 5, 515), (129, 12, 515), (136, 140, 700)):
        p = Problem(prec, hidden, tokens, vocab, pad=pad, off=off, alpha=0.7, masked=0.3, seed=pad * 10 + off)
        p.check_forward()
        p.check_backward(pad_out=pad, off_out=off, beta=0.5)
        p.check_backward(pad_out=0, off_out=0)


@pytest.mark.parametrize("prec", ["s", "b"])
@pytest.mark.parametrize("tokens", [1, 6, 150, 1100])
@pytest.mark.parametrize("masked", [0.5, 0.97, 1.0])
def test_rows_without_a_target(prec, tokens, masked):
    """Labels that are `ignore`, negative or past the vocabulary; those rows of X, lse and the gradients hold NaN and
    infinities, and nothing of it reaches a result."""
    p = Problem(prec, 104, tokens, 900, masked=masked, seed=tokens)
    p.check_forward()
    p.check_backward()
    p.check_backward(beta=0.75)


@pytest.mark.parametrize("prec", ["s", "b"])
@pytest.mark.parametrize("labels", [[3], [127, 128], [0, 255, 256, 899]])
def test_many_tokens_of_one_label(prec, labels):
    import torch
    p = Problem(prec, 328, 700, 900, seed=31, masked=0.1)
    has = xent_ref.valid(p.label, p.V, IGNORE)
    p.label[has] = np.resize(np.array(labels), int(has.sum()))
    p.dlabel = torch.from_numpy(p.label.astype(np.int32)).cuda()
    p.check_forward()
    p.check_backward(beta=0.5)


@pytest.mark.parametrize("prec", ["s", "b"])
def test_confident_and_equal_gradients(prec):
    """Every token's loss has the same gradient, and some labels take nearly all of the softmax: what rounding takes from
    their elements is the same for all tokens and would not average out."""
    p = Problem(prec, 256, 300, 1000, seed=32, spread=4.0)
    p.gloss[:] = 1.0 / 300
    p.check_forward()
    p.check_backward(glse=False)


@pytest.mark.parametrize("alpha", [-0.8, 0.0])
@pytest.mark.parametrize("tokens", [3, 140])
def test_scale_of_the_logits_may_be_negative_or_zero(alpha, tokens):
    for prec in "sb":
        p = Problem(prec, 96, tokens, 777, seed=33, alpha=alpha)
        p.check_forward()
        p.check_backward()


@pytest.mark.parametrize("prec", ["s", "b"])
def test_ignore_may_be_a_row_of_the_classifier(prec):
    import torch
    p = Problem(prec, 64, 40, 50, seed=9)
    label = p.label.copy()
    label[::3] = 7
    p.dlabel = torch.from_numpy(label.astype(np.int32)).cuda()
    loss, lse = blas.gpu_xent(prec, p.H, p.T, p.V, 1.0, p.W, p.ldW, p.X, p.ldX, p.dlabel, 7)
    got = loss.double().cpu().numpy()
    want, _, _, bound = xent_ref.forward(p.w64, p.x64, label, 1.0, 7, prec)
    assert (got[label == 7] == 0).all() and (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("prec", ["s", "b"])
@pytest.mark.parametrize("tokens", [3, 20, 140])
def test_pieces_of_the_vocabulary(prec, tokens):
    p = Problem(prec, 200, tokens, 1500, seed=11, masked=0.2)
    q = Problem(prec, 200, tokens, 1500, pad=1, seed=12, masked=0.2)        # packed
    blas.test_control(blas.TEST_XENT_PIECE, 256)
    try:
        for x in (p, q):
            x.check_forward()
            x.check_backward(beta=0.5)
            x.check_backward(glse=False, want=("X",))
            x.check_backward(want=("W",))
    finally:
        blas.test_control(blas.TEST_XENT_PIECE, 0)


@pytest.mark.parametrize("prec", ["s", "b"])
@pytest.mark.parametrize("tokens", [2, 160])
def test_large_and_infinite_logits(prec, tokens):
    import torch
    # logits of several hundreds: exp of them overflows, the result does not
    p = Problem(prec, 64, tokens, 700, alpha=300.0, seed=13)
    p.check_forward()
    p.check_backward()
    # logits of -inf take no part: a classifier row of -inf against positive hidden states
    q = Problem(prec, 64, tokens, 700, seed=14, spread=0.0)
    q.X.abs_()
    q.label[q.label == 5] = 6
    q.dlabel = torch.from_numpy(q.label.astype(np.int32)).cuda()
    q.W[5] = -float("inf")
    q.x64 = np.abs(q.x64)
    q.w64[5] = -np.inf
    q.check_forward()


@pytest.mark.parametrize("prec", ["s", "b"])
@pytest.mark.parametrize("tokens", [4, 200])
def test_same_bits_every_time_and_on_another_stream(prec, tokens):
    import torch
    p = Problem(prec, 264, tokens, 3000, seed=15, masked=0.2)
    first = p.forward()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream in (None, side.cuda_stream):
        again = p.forward(stream=stream)
        assert all(np.array_equal(a, b) for a, b in zip(first, again))
    a, b = p.check_backward(), p.check_backward()
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_nothing_to_do():
    import torch
    W = torch.randn(20, 8, device="cuda")
    none = torch.empty(0, device="cuda")
    labels = torch.empty(0, dtype=torch.int32, device="cuda")
    loss, lse = blas.gpu_xent("s", 8, 0, 20, 1.0, W, 8, none, 8, labels)
    assert loss.numel() == 0 and lse.numel() == 0
    # no tokens: gW is beta times what it was, or zeros
    gW = torch.ones(20, 8, device="cuda")
    blas.gpu_xent_grad("s", 8, 0, 20, 1.0, W, 8, none, 8, labels, IGNORE, none, none, None, 0.5, gW, 8, none, 8)
    assert (gW == 0.5).all()
    gW.fill_(float("nan"))
    blas.gpu_xent_grad("s", 8, 0, 20, 1.0, W, 8, none, 8, labels, IGNORE, none, none, None, 0.0, gW, 8, none, 8)
    assert (gW == 0).all()


@pytest.mark.parametrize("prec", ["s", "b"])
def test_training_step_captured_and_replayed(prec):
    """Loss, gradients, their norm and clipping in one graph, replayed on new inputs with eager work in between, each
    replay against the same calls made eagerly; then the chain against 64 bits."""
    import torch
    dt = {"s": torch.float32, "b": torch.bfloat16}[prec]
    H, T, V = 320, 180, 2100
    W = (torch.randn(V, H, device="cuda") * 2 / H ** 0.5).to(dt)
    X = torch.randn(T, H, device="cuda").to(dt)
    label = torch.randint(0, V, (T,), device="cuda", dtype=torch.int32)
    gloss = torch.full((T,), 1.0, device="cuda")
    gW, gX = torch.empty_like(W), torch.empty_like(X)
    loss, lse, norm = torch.empty(T, device="cuda"), torch.empty(T, device="cuda"), torch.empty(1, device="cuda")
    bias = torch.randn(777, device="cuda")
    group = blas.TensorGroup([gW, gX])
    out = blas.TensorGroup([torch.empty_like(gW), torch.empty_like(gX)])
    work = torch.empty(max(blas.xent_worksize(prec, H, T, V), blas.xent_grad_worksize(prec, H, T, V)), dtype=torch.uint8,
                       device="cuda")
    nwork = torch.empty(blas.gnrm2_worksize(group), dtype=torch.uint8, device="cuda")

    def step():
        blas.gpu_xent(prec, H, T, V, 1.0, W, H, X, H, label, IGNORE, loss, lse, work=work)
        blas.gpu_xent_grad(prec, H, T, V, 1.0, W, H, X, H, label, IGNORE, lse, gloss, None, 0.0, gW, H, gX, H, work=work)
        blas.gpu_gnrm2(group, norm, work=nwork)
        blas.gpu_gclip(group, norm, 0.5, out=out)

    results = [loss, lse, gW, gX, norm] + out.tensors
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for rep in range(4):
        X.copy_(torch.randn(T, H, device="cuda"))
        label.copy_(torch.randint(0, V, (T,), device="cuda"))
        label[::rep + 2] = IGNORE
        step()
        torch.cuda.synchronize()
        want = [x.clone() for x in results]
        for x in results:
            x.fill_(float("nan"))
        (bias * 2).sum().item()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(results, want):
            assert torch.equal(a, b), rep
    # the chain: what clipping returns has the norm asked for, and the norm is that of the gradients
    n64 = sum(float(x.double().square().sum()) for x in (gW, gX)) ** 0.5
    assert n64 > 0.5
    assert abs(float(norm) - n64) <= 4 * 2.0 ** -24 * n64
    half = xent_ref.half_step(prec)
    for x, y in zip((gW, gX), out.tensors):
        want = x.double() * (0.5 / n64)
        assert ((y.double() - want).abs() <= (half + 8 * 2.0 ** -24) * want.abs() + 2.0 ** -133).all()
    w64, x64 = W.double().cpu().numpy(), X.double().cpu().numpy()
    lab = label.cpu().numpy()
    wloss, wlse, blse, bloss = xent_ref.forward(w64, x64, lab, 1.0, IGNORE, prec)
    assert (np.abs(loss.double().cpu().numpy() - wloss) <= bloss).all()
    wW, wX, bW, bX = xent_ref.backward(w64, x64, lab, 1.0, IGNORE, lse.double().cpu().numpy(), np.ones(T), None, prec)
    assert (np.abs(gW.double().cpu().numpy() - wW) <= bW).all()
    assert (np.abs(gX.double().cpu().numpy() - wX) <= bX).all()


@pytest.mark.parametrize("prec", ["s", "b"])
def test_two_calls_at_once(prec):
    """Two streams, a workspace each: both get what a call by itself gets."""
    import torch
    ps = [Problem(prec, 256, t, 4000, seed=20 + t) for t in (9, 400)]
    want = [p.forward() for p in ps]
    streams = [torch.cuda.Stream() for _ in ps]
    works = [p.work(blas.xent_worksize(prec, p.H, p.T, p.V)) for p in ps]
    torch.cuda.synchronize()
    for _ in range(3):
        got = [blas.gpu_xent(prec, p.H, p.T, p.V, p.alpha, p.W, p.ldW, p.X, p.ldX, p.dlabel, IGNORE, work=w,
                             stream=s.cuda_stream) for p, s, w in zip(ps, streams, works)]
        torch.cuda.synchronize()
        for (l, e), (wl, we) in zip(got, want):
            assert np.array_equal(l.double().cpu().numpy(), wl) and np.array_equal(e.double().cpu().numpy(), we)


@pytest.mark.parametrize("prec", ["s", "b"])
def test_most_tokens(prec):
    """As many tokens as a call takes: offsets of P pass 32 bits.  All but 2000 of them have gradient 0, so that these
    (the first and the last ones among them) are all that a result holds."""
    import torch
    H, T, V = 12, 1 << 23, 300
    dt = {"s": torch.float32, "b": torch.bfloat16}[prec]
    gen = torch.Generator("cuda").manual_seed(3)
    X = torch.randn(T, H, generator=gen, device="cuda").to(dt)
    W = torch.randn(V, H, generator=gen, device="cuda").to(dt)
    label = torch.randint(0, V, (T,), generator=gen, device="cuda", dtype=torch.int32)
    label[1000:T // 2:7] = IGNORE
    loss, lse = blas.gpu_xent(prec, H, T, V, 1.0, W, H, X, H, label)
    torch.cuda.synchronize()
    assert torch.isfinite(loss).all() and torch.isfinite(lse).all() and (loss[label == IGNORE] == 0).all()
    some = torch.cat([torch.arange(500), torch.arange(T // 2 - 500, T // 2 + 500), torch.arange(T - 500, T)])
    at = some.cuda()
    w64, x64, y = W.double().cpu().numpy(), X[at].double().cpu().numpy(), label[at].cpu().numpy()
    wloss, wlse, blse, bloss = xent_ref.forward(w64, x64, y, 1.0, IGNORE, prec)
    assert (np.abs(lse[at].double().cpu().numpy() - wlse) <= blse).all()
    assert (np.abs(loss[at].double().cpu().numpy() - wloss) <= bloss).all()
    gloss = torch.zeros(T, device="cuda")
    gloss[at] = torch.randn(len(some), generator=gen, device="cuda")
    gW, gX = torch.full_like(W, float("nan")), torch.full_like(X, float("nan"))
    blas.gpu_xent_grad(prec, H, T, V, 1.0, W, H, X, H, label, IGNORE, lse, gloss, None, 0.0, gW, H, gX, H)
    torch.cuda.synchronize()
    wW, wX, bW, bX = xent_ref.backward(w64, x64, y, 1.0, IGNORE, lse[at].double().cpu().numpy(),
                                       gloss[at].double().cpu().numpy(), None, prec)
    assert (np.abs(gW.double().cpu().numpy() - wW) <= bW).all()
    assert (np.abs(gX[at].double().cpu().numpy() - wX) <= bX).all()
    gX[at] = 0
    assert (gX == 0).all()


@pytest.mark.parametrize("prec", ["s", "b"])
@pytest.mark.parametrize("tokens", [3, 20, 90])
def test_classifier_past_32_bits(prec, tokens):
    """W and gW of more than 2^31 elements.  Only 600 rows of W, the first and the last ones among them, are near the
    hidden states; the other logits are 0, and so are the other rows of gW but for softmax's share of them."""
    import torch
    H, V = 2056, 1100003
    dt = {"s": torch.float32, "b": torch.bfloat16}[prec]
    gen = torch.Generator("cuda").manual_seed(tokens)
    W = torch.zeros(V, H, dtype=dt, device="cuda")
    some = torch.cat([torch.arange(200), torch.arange(V // 2, V // 2 + 200), torch.arange(V - 200, V)])
    at = some.cuda()
    W[at] = (torch.randn(600, H, generator=gen, device="cuda") * 0.05).to(dt)
    pick = torch.randint(0, 600, (tokens,), generator=gen, device="cuda")
    pick[0], pick[1] = 599, 0
    label = at[pick].int()
    X = (torch.randn(tokens, H, generator=gen, device="cuda") + 30 * W[label.long()].float()).to(dt)
    loss, lse = blas.gpu_xent(prec, H, tokens, V, 1.0, W, H, X, H, label)
    torch.cuda.synchronize()
    w64, x64, y = W[at].double().cpu().numpy(), X.double().cpu().numpy(), pick.cpu().numpy()
    # the reference in 64 bits: the rows of zeros add exp(0) each to the sum and nothing to the products
    z = x64 @ w64.T
    top = np.maximum(z.max(axis=1), 0)
    want = top + np.log(np.exp(z - top[:, None]).sum(axis=1) + (V - 600) * np.exp(-top))
    dz = (H + 2) * xent_ref.U * (np.abs(x64) @ np.abs(w64).T)
    # the bound of the reference, with the tiles of all of V
    blse = dz.max(axis=1) + (128 + 8 + -(-V // 128) + 4) * xent_ref.U + 4 * xent_ref.U * np.abs(want)
    got = lse.double().cpu().numpy()
    assert (np.abs(got - want) <= blse).all(), np.abs(got - want) / blse
    wloss, k = want - z[np.arange(tokens), y], np.arange(tokens)
    assert (np.abs(loss.double().cpu().numpy() - wloss) <= blse + dz[k, y] + 2 * xent_ref.U * np.abs(wloss)).all()
    gloss = torch.randn(tokens, generator=gen, device="cuda")
    gW, gX = torch.full((V, H), float("nan"), dtype=dt, device="cuda"), torch.full_like(X, float("nan"))
    blas.gpu_xent_grad(prec, H, tokens, V, 1.0, W, H, X, H, label, IGNORE, lse, gloss, None, 0.0, gW, H, gX, H)
    torch.cuda.synchronize()
    g64 = gloss.double().cpu().numpy()
    wW, wX, bW, bX = xent_ref.backward(w64, x64, y, 1.0, IGNORE, got, g64, None, prec)
    assert (np.abs(gW[at].double().cpu().numpy() - wW) <= bW).all()
    # sums over V terms, all but 600 of them 0 (an addition of 0 rounds nothing)
    assert (np.abs(gX.double().cpu().numpy() - wX) <= bX).all()
    # the rows between: one value a column, sum_t gloss_t exp(-lse_t) x_t
    share = (g64 * np.exp(-got)) @ x64
    size = (np.abs(g64) * np.exp(-got)) @ np.abs(x64)
    v = xent_ref.half_step(prec)
    # P: 8 u and 2 u |lse| of itself and its rounding; the sum; the result's rounding
    e = size * ((8 + 4 * np.abs(got).max() + tokens + 8) * xent_ref.U + v)
    bound = torch.from_numpy(e + v * (np.abs(share) + e) + 2.0 ** -126).cuda()
    share = torch.from_numpy(share).cuda()
    for a, b in ((200, V // 2), (V // 2 + 200, V - 200)):
        for r in range(a, b, 1 << 16):
            assert ((gW[r:min(r + (1 << 16), b)].double() - share).abs() <= bound).all(), r


@pytest.mark.parametrize("prec", ["s", "b"])
def test_more_tiles_than_a_launch_takes(prec):
    """Tokens times vocabulary beyond 2^36: the forward product goes out in several launches (here two, from row 32512
    on).  Half of the labels and most of the softmax are in the rows of the second one."""
    import torch
    H, T, V = 8, (1 << 21) + 3, 33000
    dt = {"s": torch.float32, "b": torch.bfloat16}[prec]
    gen = torch.Generator("cuda").manual_seed(7)
    X = torch.randn(T, H, generator=gen, device="cuda").to(dt)
    W = torch.randn(V, H, generator=gen, device="cuda")
    W[32512:] *= 3.0
    W = W.to(dt)
    label = torch.randint(0, V, (T,), generator=gen, device="cuda", dtype=torch.int32)
    label[::2] = torch.randint(32512, V, ((T + 1) // 2,), generator=gen, device="cuda", dtype=torch.int32)
    loss, lse = blas.gpu_xent(prec, H, T, V, 1.0, W, H, X, H, label)
    torch.cuda.synchronize()
    at = torch.cat([torch.arange(200), torch.arange(T // 2 - 100, T // 2 + 100), torch.arange(T - 200, T)]).cuda()
    w64, x64, y = W.double().cpu().numpy(), X[at].double().cpu().numpy(), label[at].cpu().numpy()
    wloss, wlse, blse, bloss = xent_ref.forward(w64, x64, y, 1.0, IGNORE, prec)
    off = [float((np.abs(got[at].double().cpu().numpy() - want) / bound).max())
           for got, want, bound in ((lse, wlse, blse), (loss, wloss, bloss))]
    assert max(off) <= 1, off


def busy():
    """Tens of milliseconds of work on the current stream."""
    import torch
    a = torch.ones(8192, 8192, device="cuda")
    for _ in range(4):
        a = a @ a * 2.0 ** -13
    return a


@pytest.mark.parametrize("prec", ["s", "b"])
@pytest.mark.parametrize("tokens", [4, 300])
@pytest.mark.parametrize("to_default", [False, True])
def test_another_stream_comes_after_the_current_one(prec, tokens, to_default):
    """Operands and workspaces that the current stream is still filling, and new memory whose last user is still at
    work there: a call on another stream comes after both."""
    import torch
    p = Problem(prec, 264, tokens, 3000, seed=41, masked=0.2)
    H, T, V = p.H, p.T, p.V
    f = [torch.from_numpy(a).cuda() for a in (p.gloss, p.glse)]
    X, label = p.X.contiguous(), p.dlabel
    sizes = [blas.xent_worksize(prec, H, T, V), blas.xent_grad_worksize(prec, H, T, V)]

    def step(X, label, out, works, stream):
        loss, lse = blas.gpu_xent(prec, H, T, V, 1.0, p.W, p.ldW, X, H, label, IGNORE, *out[:2], work=works[0], stream=stream)
        gW, gX = blas.gpu_xent_grad(prec, H, T, V, 1.0, p.W, p.ldW, X, H, label, IGNORE, lse, *f, 0.0, out[2], H, out[3], H,
                                    work=works[1], stream=stream)
        norm = blas.gpu_gnrm2([gW, gX], out[4], work=works[2], stream=stream)
        blas.gpu_gclip([gW, gX], norm, 0.5 * scale, stream=stream)
        return [loss, lse, gW, gX, norm]

    def fresh():
        return [None, None, torch.empty(V, H, dtype=X.dtype, device="cuda"),
                torch.empty(T, H, dtype=X.dtype, device="cuda"), None]

    scale = 1.0
    scale = float(step(X, label, fresh(), [None] * 3, None)[4])
    want = step(X, label, fresh(), [None] * 3, None)
    torch.cuda.synchronize()
    first, second = torch.cuda.current_stream(), torch.cuda.Stream()
    current, other = (second, first) if to_default else (first, second)
    with torch.cuda.stream(current):
        for given in (True, False):
            late_x, late_label = torch.full_like(X, float("nan")), torch.full_like(label, IGNORE)
            out, works = fresh(), [None] * 3
            torch.cuda.synchronize()
            busy()
            late_x.copy_(X)
            late_label.copy_(label)
            if given:
                out = [torch.full_like(x, float("nan")) for x in want]
                works = [p.work(n) for n in sizes] + [p.work(blas.gnrm2_worksize(want[2:4]))]
            else:               # memory of these sizes goes back to the allocator while it is still to be written
                for n in sizes + [4 * T] * 2 + [blas.gnrm2_worksize(want[2:4])]:
                    p.work(n)
            got = step(late_x, late_label, out, works, other.cuda_stream)
            other.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b)
            torch.cuda.synchronize()


@pytest.mark.parametrize("prec", ["s", "b"])
def test_another_stream_inside_a_capture(prec):
    """A second stream of the same capture, with and without new memory; a stream outside gets no new memory."""
    import torch
    p = Problem(prec, 264, 70, 3000, seed=42, masked=0.2)
    H, T, V = p.H, p.T, p.V
    X, label = p.X.contiguous(), p.dlabel
    loss, lse = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
    work = p.work(blas.xent_worksize(prec, H, T, V))
    side, outside = torch.cuda.Stream(), torch.cuda.Stream()

    def call(stream, *given, work=None):
        return blas.gpu_xent(prec, H, T, V, 1.0, p.W, p.ldW, X, H, label, IGNORE, *given, work=work, stream=stream)

    call(None, loss, lse, work=work)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        side.wait_stream(torch.cuda.current_stream())
        call(side.cuda_stream, loss, lse, work=work)
        loss2, lse2 = call(side.cuda_stream)
        with pytest.raises(ValueError, match="captured"):
            call(outside.cuda_stream)
        torch.cuda.current_stream().wait_stream(side)
        total = loss + loss2
    for seed in range(4):
        label.copy_(torch.randint(0, V, (T,), device="cuda"))
        X.copy_(torch.randn(T, H, device="cuda"))
        wloss, wlse = call(None)
        torch.cuda.synchronize()
        for x in (loss, lse, loss2, lse2, total):
            x.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        for a, b in ((loss, wloss), (lse, wlse), (loss2, wloss), (lse2, wlse), (total, 2 * wloss)):
            assert torch.equal(a, b), seed


@pytest.mark.parametrize("prec", ["s", "b"])
@pytest.mark.parametrize("tokens", [5, 90])
def test_gradients_between_the_rows_of_the_operands(prec, tokens):
    """X beside gX and W beside gW in the halves of wide matrices, loss beside lse: no memory is shared."""
    import torch
    p = Problem(prec, 200, tokens, 1300, seed=51, masked=0.2)
    H, T, V = p.H, p.T, p.V
    f = [torch.from_numpy(a).cuda() for a in (p.gloss, p.glse)]
    want = list(blas.gpu_xent(prec, H, T, V, 1.0, p.W, p.ldW, p.X, p.ldX, p.dlabel, IGNORE))
    gW, gX = torch.empty(V, H, dtype=p.W.dtype, device="cuda"), torch.empty(T, H, dtype=p.W.dtype, device="cuda")
    want += blas.gpu_xent_grad(prec, H, T, V, 1.0, p.W, p.ldW, p.X, p.ldX, p.dlabel, IGNORE, want[1], *f, 0.0, gW, H, gX, H)
    wide = torch.zeros(V + 1, 2 * H, dtype=gW.dtype, device="cuda")
    w, x, both = wide[:V], torch.zeros_like(gX).repeat(1, 3), torch.empty(2 * T, device="cuda")
    w[:, H:], x[:, H:2 * H] = p.W, p.X
    got = list(blas.gpu_xent(prec, H, T, V, 1.0, w[:, H:], 2 * H, x[:, H:], 3 * H, p.dlabel, IGNORE, both[:T], both[T:]))
    got += blas.gpu_xent_grad(prec, H, T, V, 1.0, w[:, H:], 2 * H, x[:, H:], 3 * H, p.dlabel, IGNORE, got[1], *f, 0.0,
                              w, 2 * H, x, 3 * H)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a[:, :H] if a.dim() == 2 else a, b)
    assert torch.equal(w[:, H:].float().nan_to_num(), p.W.float().nan_to_num()) and (x[:, 2 * H:] == 0).all()
    for off in (1, 2 * H - 1):          # one element of every row too far
        with pytest.raises(blas.GpuError, match="overlaps"):
            blas.gpu_xent_grad(prec, H, T, V, 1.0, w[:, H:], 2 * H, x[:, H:], 3 * H, p.dlabel, IGNORE, got[1], *f, 0.0,
                               wide.view(-1)[off:], 2 * H, None, H)
    with pytest.raises(blas.GpuError, match="overlaps"):
        blas.gpu_xent(prec, H, T, V, 1.0, p.W, p.ldW, p.X, p.ldX, p.dlabel, IGNORE, both[:T], both[T - 1:2 * T - 1])


@pytest.mark.parametrize("prec", ["s", "b"])
@pytest.mark.parametrize("pad", [0, 1])
def test_nothing_behind_the_workspace_is_written(prec, pad):
    """Vocabularies that end in every part of a tile, on both sides of the sizes at which the tiles change."""
    import torch
    for tokens in (1, 32, 33, 257, 600):
        for vocab in (1, 127, 129, 257, 1025, 2000):
            p = Problem(prec, 72, tokens, vocab, pad=pad, seed=tokens + vocab)
            sizes = [f(prec, 72, tokens, vocab) for f in (blas.xent_worksize, blas.xent_grad_worksize)]
            works = [torch.full((size + 4096,), 0x5a, dtype=torch.uint8, device="cuda") for size in sizes]
            gW, gX = (torch.empty(n, 72, dtype=p.W.dtype, device="cuda") for n in (vocab, tokens))
            loss, lse = blas.gpu_xent(prec, 72, tokens, vocab, 1.0, p.W, p.ldW, p.X, p.ldX, p.dlabel, work=works[0])
            blas.gpu_xent_grad(prec, 72, tokens, vocab, 1.0, p.W, p.ldW, p.X, p.ldX, p.dlabel, IGNORE, lse,
                               torch.ones(tokens, device="cuda"), None, 0.0, gW, 72, gX, 72, work=works[1])
            torch.cuda.synchronize()
            for work, size in zip(works, sizes):
                assert (work[size:] == 0x5a).all(), (tokens, vocab)
            p.check_forward()
