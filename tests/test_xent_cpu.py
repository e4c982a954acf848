"""The cross entropy's formulas against differences, and what its entry points (and those of the group norm and
clipping) refuse, without a device: every refusal is made on the host before anything is launched."""
import ctypes as C

import numpy as np
import pytest

import xent_ref
from ulmblas_amd import blas, lib

BAD = 1


def test_formula_against_differences():
    rng = np.random.default_rng(1)
    V, T, H, alpha = 23, 9, 7, 0.7
    W, X = rng.standard_normal((V, H)), rng.standard_normal((T, H))
    label = rng.integers(0, V, T)
    label[[2, 5]] = [-100, V]
    gloss, glse = rng.standard_normal(T), rng.standard_normal(T)

    def value(W, X):
        loss, lse, _, _ = xent_ref.forward(W, X, label, alpha, -100, "s")
        return gloss @ loss + glse @ lse

    _, lse, _, _ = xent_ref.forward(W, X, label, alpha, -100, "s")
    gW, gX, _, _ = xent_ref.backward(W, X, label, alpha, -100, lse, gloss, glse, "s")
    h = 1e-5
    for name, A, g in (("W", W, gW), ("X", X, gX)):
        for _ in range(5):
            d = rng.standard_normal(A.shape)
            up, down = (value(W + h * d, X), value(W - h * d, X)) if name == "W" else (value(W, X + h * d), value(W, X - h * d))
            # h^2/6 times a third derivative of order |d|^3 ~ (VH)^1.5, and rounding 2^-53 |value| / h
            assert abs((up - down) / (2 * h) - (g * d).sum()) < 1e-6, name


P = C.c_void_p(4096)        # a pointer that nothing follows: the refusals come first


def xent(p, hidden=8, tokens=4, vocab=10, ldW=8, ldX=8, W=P, X=P, label=P, loss=P, lse=P, work=P):
    return getattr(lib.load(), f"ulmblas_gpu_{p}xent")(hidden, tokens, vocab, 1.0, W, ldW, X, ldX, label, -100, loss, lse,
                                                       work, None)


def grad(p, hidden=8, tokens=4, vocab=10, ldW=8, ldX=8, ldGW=8, ldGX=8, W=P, X=P, label=P, lse=P, gloss=P, gW=P, gX=P,
         work=P):
    return getattr(lib.load(), f"ulmblas_gpu_{p}xent_grad")(hidden, tokens, vocab, 1.0, W, ldW, X, ldX, label, -100, lse,
                                                            gloss, None, 0.0, gW, ldGW, gX, ldGX, work, None)


@pytest.mark.parametrize("p", ["s", "b"])
def test_refusals_of_the_cross_entropy(p):
    for kw in (dict(hidden=0, ldW=8), dict(hidden=-1), dict(hidden=(1 << 20) + 1, ldW=1 << 21, ldX=1 << 21), dict(tokens=-1),
               dict(tokens=(1 << 23) + 1), dict(vocab=0), dict(vocab=(1 << 28) + 1), dict(ldW=7), dict(ldX=7), dict(ldW=1 << 21),
               dict(W=None), dict(X=None), dict(label=None), dict(loss=None), dict(lse=None), dict(work=None), dict(work=C.c_void_p(4104))):
        assert xent(p, **kw) == BAD, kw
        assert lib.load().ulmblas_gpu_last_error() != b""
    for kw in (dict(hidden=0), dict(tokens=-1), dict(vocab=0), dict(ldW=7), dict(ldX=7), dict(ldGW=7), dict(ldGX=7),
               dict(ldW=1 << 21), dict(W=None), dict(X=None), dict(label=None), dict(lse=None), dict(gloss=None), dict(work=None),
               dict(work=C.c_void_p(4104))):
        assert grad(p, **kw) == BAD, kw
    odd = C.c_void_p(4097)
    for kw in (dict(W=odd), dict(X=odd), dict(label=odd), dict(loss=odd), dict(lse=odd)):
        assert xent(p, **kw) == BAD, kw
    for kw in (dict(W=odd), dict(X=odd), dict(label=odd), dict(lse=odd), dict(gloss=odd), dict(gW=odd), dict(gX=odd)):
        assert grad(p, **kw) == BAD, kw
    # nothing to do: no device is needed
    assert xent(p, tokens=0, W=None, X=None, label=None, loss=None, lse=None, work=None) == 0
    assert grad(p, gW=None, gX=None) == 0


@pytest.mark.parametrize("p", ["s", "b"])
def test_worksizes(p):
    for bad in ((0, 1, 1), (1, -1, 1), (1, 1, 0), ((1 << 20) + 1, 1, 1)):
        for f in (blas.xent_worksize, blas.xent_grad_worksize):
            with pytest.raises(blas.GpuError):
                f(p, *bad)
    # the gradient keeps a piece of the vocabulary, never the logits: P, a packed piece of W and sums of gX
    size = {"s": 4, "b": 2}[p]
    big = blas.xent_grad_worksize(p, 4096, 1 << 16, 1 << 18)
    assert big < (1 << 16) * (1 << 18) * size
    # no tokens need what their bookkeeping takes, no more
    assert blas.xent_worksize(p, 8, 0, 10) > 0 and blas.xent_grad_worksize(p, 8, 0, 10) > 0
    # the largest sizes are counted in 64 bits
    assert blas.xent_worksize(p, 1 << 20, 1 << 23, 1 << 28) > 1 << 40


def group(count=2, type=b"sb", n=(4, 4), x=(4096, 4096), y=(4096, 4096), norm=P, work=P, largest=1.0, which="norm"):
    L = lib.load()
    lengths = (C.c_long * 2)(*n) if n else None
    px = (C.c_void_p * 2)(*x) if x else None
    py = (C.c_void_p * 2)(*y) if y else None
    if which == "norm":
        return L.ulmblas_gpu_gnrm2(count, type, lengths, px, norm, work, None)
    return L.ulmblas_gpu_gclip(count, type, lengths, px, py, norm, largest, None)


def test_refusals_of_the_group():
    for which in ("norm", "clip"):
        for kw in (dict(count=-1), dict(type=b"sd"), dict(type=None), dict(n=None), dict(x=None), dict(n=(-1, 4)),
                   dict(n=((1 << 40) + 1, 4)), dict(x=(None, 4096)), dict(x=(4098, 4096)), dict(x=(4096, 4097)),
                   dict(norm=None)):
            assert group(which=which, **kw) == BAD, (which, kw)
    assert group(work=None) == BAD and group(work=C.c_void_p(4100)) == BAD
    for kw in (dict(largest=-1.0), dict(largest=float("nan")), dict(y=None), dict(y=(4098, 4096)), dict(y=(None, 4096))):
        assert group(which="clip", **kw) == BAD, kw
    assert group(which="clip", count=0, norm=None) == 0
    # what is written overlaps nothing but its own tensor: 4 fp32 and 4 bf16 elements are 16 and 8 bytes
    for kw in (dict(y=(4096, 4096)), dict(x=(4096, 4200), y=(4096, 4108)), dict(x=(4096, 4200), y=(4300, 4110)),
               dict(x=(4096, 4200), y=(4100, 4200)), dict(x=(4096, 4200), y=(4196, 4300))):
        assert group(which="clip", **kw) == BAD, kw
        assert b"overlaps" in lib.load().ulmblas_gpu_last_error(), kw


def test_wrappers_refuse_what_does_not_fit():
    torch = pytest.importorskip("torch")
    W, X = torch.zeros(10, 8), torch.zeros(4, 8)
    label = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="not on a GPU"):
        blas.gpu_xent("s", 8, 4, 10, 1.0, W, 8, X, 8, label)
    with pytest.raises(ValueError, match="window"):
        blas.gpu_xent("s", 8, 4, 11, 1.0, W, 8, X, 8, label)
    with pytest.raises(ValueError, match="window"):
        blas.gpu_xent("s", 8, 4, 10, 1.0, W, 8, X, 9, label)
    with pytest.raises(TypeError, match="W must be"):
        blas.gpu_xent("b", 8, 4, 10, 1.0, W, 8, X, 8, label)
    with pytest.raises(TypeError, match="labels"):
        blas.gpu_xent("s", 8, 4, 10, 1.0, W, 8, X, 8, label.long())
    with pytest.raises(ValueError, match="labels"):
        blas.gpu_xent("s", 8, 4, 10, 1.0, W, 8, X, 8, label[:3])
    f = torch.zeros(4)
    with pytest.raises(ValueError, match="gW"):
        blas.gpu_xent_grad("s", 8, 4, 10, 1.0, W, 8, X, 8, label, -100, f, f, None, 0.0, torch.zeros(9, 8), 8, None, 8)
    with pytest.raises(ValueError, match="lse"):
        blas.gpu_xent_grad("s", 8, 4, 10, 1.0, W, 8, X, 8, label, -100, f[:2], f, None, 0.0, None, 8, None, 8)
    with pytest.raises(TypeError, match="tensor 1"):
        blas.TensorGroup([f, f.double()])
    with pytest.raises(ValueError, match="contiguous"):
        blas.TensorGroup([torch.zeros(4, 4).T])
    with pytest.raises(ValueError, match="not on a GPU"):
        blas.TensorGroup([f])


class FakeStreams:
    """torch's streams and allocator as far as the wrappers use them: a log of what they do, in order."""

    def __init__(self, monkeypatch, captured=()):
        torch = pytest.importorskip("torch")
        self.log, self.now, fake = [], 7, self

        class Stream:
            def __init__(self, raw, device=None):
                self.cuda_stream = raw or "a new one"

            def wait_stream(self, other):
                fake.log.append(f"{self.cuda_stream} waits for {other.cuda_stream}")

        default = Stream(1)
        default.cuda_stream = 0

        class Inside:
            def __init__(self, stream):
                self.stream = stream

            def __enter__(self):
                self.before, fake.now = fake.now, self.stream.cuda_stream

            def __exit__(self, *exc):
                fake.now = self.before

        class Tensor:
            def record_stream(self, stream):
                fake.log.append(f"kept for {stream.cuda_stream}")

            def __getitem__(self, key):
                return self

        def empty(n, **kw):
            fake.log.append(f"memory of {fake.now}")
            return Tensor()

        for name, value in (("current_device", lambda: 0), ("current_stream", lambda *a: Stream(fake.now)),
                            ("ExternalStream", Stream), ("default_stream", lambda *a: default), ("stream", Inside),
                            ("is_current_stream_capturing", lambda: fake.now in captured)):
            monkeypatch.setattr(torch.cuda, name, value)
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: fake.now)
        monkeypatch.setattr(torch, "empty", empty)
        monkeypatch.setattr(torch, "zeros", empty)
        self.device = torch.device("cuda", 0)
        self.dtype = torch.uint8


def test_another_stream_waits_before_memory_is_handed_out(monkeypatch):
    """The allocator hands out memory in the current stream's order: another stream has to wait for that one first."""
    f = FakeStreams(monkeypatch)
    with blas._On(f.device, 11) as on:
        assert on.stream == 11
        on.empty(5, f.dtype)
    assert f.log == ["11 waits for 7", "memory of 7", "kept for 11"]
    f.log.clear()
    with blas._On(f.device, 0) as on:           # the default stream
        assert on.stream == 0
        on.empty(5, f.dtype)
    assert f.log == ["0 waits for 7", "memory of 7", "kept for 0"]
    for given in (None, 7):
        f.log.clear()
        with blas._On(f.device, given) as on:
            assert on.stream == 7
            on.empty(5, f.dtype)
        assert f.log == ["memory of 7"]


@pytest.mark.parametrize("captured", [(7,), (11,), (7, 11)])
def test_another_stream_of_a_capture(monkeypatch, captured):
    f = FakeStreams(monkeypatch, captured)
    with blas._On(f.device, 11) as on:
        if len(captured) == 2:
            on.empty(5, f.dtype)
            assert f.log == ["11 waits for 7", "memory of 7", "kept for 11"]
        else:                           # nothing can wait across a capture's border: no new memory, no order
            with pytest.raises(ValueError, match="captured"):
                on.empty(5, f.dtype)
            assert f.log == ["memory of 7"] and on.stream == 11


def test_another_stream_of_the_other_calls_with_new_memory(monkeypatch):
    """LU and the complex product: pivots, status and workspace are filled and handed out before the stream waits."""
    torch = pytest.importorskip("torch")
    A = torch.zeros(8, 8, dtype=torch.float64)
    f = FakeStreams(monkeypatch)

    class Library:
        def __getattr__(self, name):
            if name.endswith("worksize"):
                return lambda *a: 64
            return lambda *a: f.log.append(f"{name} on {a[-1]}") or 0

    library = Library()
    monkeypatch.setattr(blas, "load", lambda: library)
    monkeypatch.setattr(blas, "_dev_ptr", lambda x: None)
    blas.gpu_dgetrf(8, 8, A, 8, stream=11)
    assert f.log == ["memory of 7"] * 3 + ["11 waits for 7"] + ["kept for 11"] * 3 + ["ulmblas_gpu_dgetrf on 11"]
    f.log.clear()
    blas.gpu_cgemm("z", "N", "N", 2, 2, 2, 1.0, A, 2, A, 2, 0.0, A, 2, stream=11)
    assert f.log == ["memory of 7", "11 waits for 7", "kept for 11", "ulmblas_gpu_zgemm on 11"]


def have_gpu():
    return pytest.importorskip("torch").cuda.is_available()


AREA = {name: C.c_void_p((i + 1) << 44) for i, name in enumerate(("W", "X", "label", "loss", "lse", "gloss", "gW", "gX", "work"))}


def refused(call, p, **kw):
    """Whether a call on addresses that nothing follows is refused for an overlap (anything else needs a GPU)."""
    names = ("W", "X", "label", "loss", "lse", "work") if call is xent else ("W", "X", "label", "lse", "gloss", "gW", "gX", "work")
    status = call(p, **{**{n: AREA[n] for n in names}, **kw})
    text = lib.load().ulmblas_gpu_last_error()
    assert status != 0
    return status == BAD and b"overlaps" in text


@pytest.mark.parametrize("p", ["s", "b"])
def test_overlapping_operands_are_refused(p):
    size = {"s": 4, "b": 2}[p]

    def at(name, off):
        return C.c_void_p(AREA[name].value + off)

    # hidden 8, 4 tokens, 10 columns of W: the last bytes of each operand
    last = {"W": 80 * size, "X": 32 * size, "label": 16, "loss": 16, "lse": 16, "gloss": 16, "gW": 80 * size, "gX": 32 * size}
    for a in ("loss", "lse", "work"):
        for b in ("W", "X", "label", "loss", "lse"):
            if a != b:
                assert refused(xent, p, **{a: at(b, 0)}), (a, b)
                assert refused(xent, p, **{a: at(b, last[b] // 16 * 16 - 16)}), (a, b)
    assert refused(xent, p, loss=at("work", blas.xent_worksize(p, 8, 4, 10) - 4))
    for tokens in (4, 16):
        for a in ("gW", "gX", "work"):
            for b in ("W", "X", "label", "lse", "gloss", "gW", "gX"):
                if a != b:
                    assert refused(grad, p, tokens=tokens, **{a: at(b, 0)}), (a, b)
                    assert refused(grad, p, tokens=tokens, **{a: at(b, last[b] // 16 * 16 - 16)}), (a, b)
        assert refused(grad, p, tokens=tokens, gW=at("work", blas.xent_grad_worksize(p, 8, tokens, 10) - 4))
    # the gradient of lse, too
    assert lib.load()[f"ulmblas_gpu_{p}xent_grad"](8, 4, 10, C.c_float(1.0), AREA["W"], 8, AREA["X"], 8, AREA["label"], -100,
                                                   AREA["lse"], AREA["gloss"], AREA["gX"], C.c_float(0.0), AREA["gW"], 8,
                                                   AREA["gX"], 8, AREA["work"], None) == BAD


def test_windows_between_the_columns_of_others():
    """Random windows in one area: refused exactly where a written one shares an element with another."""
    if have_gpu():
        pytest.skip("the calls that are not refused would run on addresses that nothing follows")
    rng = np.random.default_rng(17)
    met = 0
    for trial in range(1500):
        H, T, V = (int(n) for n in (rng.integers(1, 5), rng.integers(1, 12), rng.integers(1, 12)))
        pitch = int(rng.integers(H, 12))
        # half the trials: all columns equally far apart, as in the parts of one wide matrix
        ld = [pitch if trial % 2 else int(rng.integers(H, 14)) for _ in range(4)]
        at = [int(rng.integers(0, 60)) for _ in range(4)]
        if trial % 3 == 0:
            at = [int(a) * H for a in rng.permutation(4)]
        columns = (V, T, V, T)
        cells = [{a + c * l + h for c in range(n) for h in range(H)} for a, l, n in zip(at, ld, columns)]
        meets = any(cells[i] & cells[j] for i in (2, 3) for j in range(4) if i != j)
        where = [C.c_void_p(AREA["W"].value + 4 * a) for a in at]
        got = refused(grad, "s", hidden=H, tokens=T, vocab=V, ldW=ld[0], ldX=ld[1], ldGW=ld[2], ldGX=ld[3], W=where[0],
                      X=where[1], gW=where[2], gX=where[3])
        assert got == meets, (H, T, V, ld, at)
        met += meets
    assert 200 < met < 1300         # both answers were asked for


def test_clipping_refuses_a_norm_inside_a_tensor_it_writes():
    """Some workgroups would read the norm after others have scaled it."""
    for off in (0, 12):
        for kw in (dict(x=(4096, 5000), y=(4096, 5000)), dict(x=(8192, 9000), y=(4096, 5000))):
            assert group(which="clip", norm=C.c_void_p(4096 + off), **kw) == BAD, (off, kw)
            assert b"overlaps" in lib.load().ulmblas_gpu_last_error()
    assert group(which="clip", n=(0, 4), x=(None, 4096), y=(None, 4096), norm=C.c_void_p(4100)) == BAD


def test_norm_refuses_a_workspace_inside_a_tensor():
    size, at = blas.gnrm2_worksize([None] * 2), 1 << 30
    # the second tensor: 4 bf16 elements from `at` on, or long enough to reach into the workspace or around it
    for kw in (dict(work=C.c_void_p(at)), dict(work=C.c_void_p(at + 8 - size)), dict(work=C.c_void_p(at + 4096), n=(4, 2049)),
               dict(work=C.c_void_p(at + 4096), n=(4, 1 << 30))):
        assert group(**{**dict(x=(1 << 40, at)), **kw}) == BAD, kw
        assert b"workspace overlaps" in lib.load().ulmblas_gpu_last_error(), kw


def test_a_group_whose_memory_was_replaced_is_refused(monkeypatch):
    """Its addresses are those of memory that may belong to others by now."""
    torch = pytest.importorskip("torch")
    monkeypatch.setattr(blas, "_device_of", lambda named: None)

    def make():
        tensors = [torch.ones(5), torch.ones(7, dtype=torch.bfloat16), torch.ones(9)]
        return tensors, blas.TensorGroup(tensors)

    norm = torch.ones(1)
    tensors, group = make()
    group.check()
    tensors[1].fill_(3.0)               # other values in the same memory are no other memory
    group.check()
    tensors[1].data = torch.ones(7, dtype=torch.bfloat16)
    tensors2, resized = make()
    tensors2[2].resize_(1 << 20)
    tensors3, released = make()
    tensors3[0].untyped_storage().resize_(0)
    for g, i in ((group, 1), (resized, 2), (released, 0)):
        for call in (lambda: blas.gpu_gnrm2(g), lambda: blas.gpu_gclip(g, norm, 1.0),
                     lambda: blas.gpu_gclip(make()[1], norm, 1.0, out=g), lambda: blas.gpu_gclip(g, norm, 1.0, out=make()[1])):
            with pytest.raises(ValueError, match=f"tensor {i} was replaced"):
                call()


def test_ignore_beyond_32_bits_is_refused():
    """As a C int 2^32 + 3 would be 3, and the tokens of row 3 would lose their target."""
    torch = pytest.importorskip("torch")
    W, X, f = torch.zeros(10, 8), torch.zeros(4, 8), torch.zeros(4)
    label = torch.zeros(4, dtype=torch.int32)
    for ignore in ((1 << 32) + 3, 1 << 31, -(1 << 31) - 1):
        with pytest.raises(ValueError, match="32-bit"):
            blas.gpu_xent("s", 8, 4, 10, 1.0, W, 8, X, 8, label, ignore)
        with pytest.raises(ValueError, match="32-bit"):
            blas.gpu_xent_grad("s", 8, 4, 10, 1.0, W, 8, X, 8, label, ignore, f, f, None, 0.0, None, 8, None, 8)
    for ignore in ((1 << 31) - 1, -(1 << 31)):          # these go on to what is wrong with the operands
        with pytest.raises(ValueError, match="not on a GPU"):
            blas.gpu_xent("s", 8, 4, 10, 1.0, W, 8, X, 8, label, ignore)


@pytest.mark.parametrize("p", ["s", "b"])
def test_workspace_of_the_forward_call(p):
    """8 bytes for every token and 128 rows of W, a copy of X (in steps of 128 bytes), for bf16 at most 128 MiB of
    packed W, and 16 bytes a token (tokens in 256s)."""
    size = {"s": 4, "b": 2}[p]
    for hidden, tokens, vocab in ((4096, 8192, 131072), (64, 1 << 20, 131072), (1000, 333, 20011), (8, 40, 300)):
        tp, hp = -(-tokens // 256) * 256, -(-hidden // (128 // size)) * 128
        packed = (1 << 27 if p == "b" else 0) + 256 * hp
        assert blas.xent_worksize(p, hidden, tokens, vocab) <= tp * (-(-vocab // 256) * 16 + hp + 16) + packed + 2048
    # what the tiles of 64 rows need, which bf16 takes up to 32 tokens where W lies off words
    assert blas.xent_worksize("b", 64, 32, 1 << 20) >= 256 * (1 << 20) // 64 * 8
