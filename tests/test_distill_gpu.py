"""The distillation loss and its gradient against fp64, over vocabularies, masks, reductions and upstreams."""
import math

import pytest
import torch

from firefly_b200 import _capi, distillation_loss
from firefly_b200.decoder import DecoderConfig, build_decoder
from oracle import distill_oracle as O

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _case(n, V, k, seed, dtype=torch.bfloat16, labels=False, tail=False, T=1.0, pad=True, spread=2.5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = torch.randn(n, V, device=DEV, generator=g) * spread
    z = s + torch.randn(n, V, device=DEV, generator=g) * 0.7
    top = torch.topk(z, min(k, V), dim=1)
    ids, t = top.indices, top.values
    lse = torch.logsumexp(z / T, 1) if tail else None
    if pad and n > 2:
        keep = torch.randint(0, k + 1, (n, 1), device=DEV, generator=g)
        keep[::3] = k
        ids = torch.where(torch.arange(ids.shape[1], device=DEV)[None] < keep, ids, torch.full_like(ids, -1))
    lab = None
    if labels:
        lab = torch.randint(0, V, (n,), device=DEV, generator=g)
        lab[1::4] = -100
        lab[::5] = ids[::5, 0].clamp(min=0)  # the teacher's first choice is the label
    return s.to(dtype), ids, t, lab, lse


def _check(s, ids, t, lab, lse, T, alpha, reduction="mean", up=1.0, grad_of=None):
    """Loss and gradient against the oracle.  The loss: log p, log q and their products carry the errors of
    fp32 exponentials, logarithms and sums (below 2^-19 of the magnitudes that are added).  A gradient element
    is factor * (q - p): 2^-18 of q + p (the exponential's argument, up to 2^6, is rounded to 2^-24 of itself),
    then one rounding to the logits' type."""
    x = s.detach().clone().requires_grad_(True) if grad_of is None else grad_of
    got = distillation_loss(x, ids, t, lab, teacher_lse=lse, temperature=T, alpha=alpha, reduction=reduction)
    s64 = s.detach().double().requires_grad_(True)
    rows, counted, scale = O.losses(s64, ids, t, lab, lse, T, alpha)
    cnt = max(1, sum(counted))
    tol = 2.0 ** -19 * (T * T * (4 + scale) + 16)
    if reduction == "none":
        assert got.shape == rows.shape
        assert bool(((got.double() - rows).abs() <= tol).all())
        u = torch.linspace(0.5, 2.0, s.shape[0], device=DEV) * up
        got.backward(u)
        (rows * u.double()).sum().backward()
        f = u.double()[:, None]
    else:
        want = rows.sum() / (cnt if reduction == "mean" else 1)
        tol = tol.sum() / (cnt if reduction == "mean" else 1) + 2.0 ** -24 * float(want.detach().abs())
        assert abs(float(got.detach()) - float(want.detach())) <= float(tol)
        (got * up).backward() if up != 1.0 else got.backward()
        (want * up).backward()
        f = up / (cnt if reduction == "mean" else 1)
    assert x.grad.dtype == s.dtype and x.grad.shape == s.shape
    want = s64.grad
    q = torch.softmax(s.double() / T, 1) + torch.softmax(s.double(), 1)
    p = torch.zeros_like(q)
    on = (ids >= 0) & (ids < s.shape[1])
    p.scatter_add_(1, torch.where(on, ids, 0).long(), on.double())
    if lab is not None:
        # the label's own term is factor * 1, and the factor (upstream * (1 - alpha) / count, each step rounded)
        # and the subtraction are off by up to four halves of 2^-23 of it
        y = torch.zeros_like(q).scatter_(1, lab.clamp(min=0)[:, None], 1.0) * (lab >= 0)[:, None]
        p = p + y * 2.0 ** -4  # 2^-18 * 2 * 2^-4 = 4 * 2^-23
    tiny = torch.finfo(s.dtype).smallest_normal * torch.finfo(s.dtype).eps
    tol = 2.0 ** -18 * f * max(T, 1) * 2 * (q + p) + torch.finfo(s.dtype).eps / 2 * want.abs() + tiny
    if lse is not None:  # off the entries: q (1 - p_rest / q_rest), with 1 - sum p off by k 2^-24
        tol = tol + 2.0 ** -18 * f * T
    off = (x.grad.double() - want).abs()
    worst = int((off / tol).argmax())
    assert bool((off <= tol).all()), (float((off / tol).max()), divmod(worst, s.shape[1]))
    live = torch.tensor(counted, device=DEV)
    assert not x.grad[~live].any()
    assert _capi.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,k", [(1, 1, 1), (1, 7, 3), (5, 100, 100), (3, 1000, 1), (9, 4099, 33), (4, 32000, 64),
                                   (2, 70001, 100), (500, 257, 20)])
def test_loss_and_gradient(n, V, k, dtype):
    s, ids, t, _, _ = _case(n, V, k, n + V)
    _check(s.to(dtype), ids, t, None, None, 1.0, 1.0)


@pytest.mark.parametrize("V", [131071, 131072, 250007])
@pytest.mark.parametrize("n", [1, 3])
def test_long_vocabularies(V, n):
    s, ids, t, lab, lse = _case(n, V, 100, V, labels=True, tail=True, pad=False)
    _check(s, ids, t, lab, lse, 1.0, 0.5)
    _check(s.float(), ids, t, None, lse, 1.0, 1.0)


@pytest.mark.parametrize("T", [1.0, 2.0, 0.7, 4.0])
@pytest.mark.parametrize("labels,alpha", [(False, 1.0), (True, 0.5), (True, 1.0), (True, 0.0), (False, 0.3)])
@pytest.mark.parametrize("tail", [False, True])
def test_temperature_labels_and_tail(T, labels, alpha, tail):
    s, ids, t, lab, lse = _case(12, 2001, 30, 3, labels=labels, tail=tail, T=T)
    for dtype in (torch.bfloat16, torch.float32):
        _check(s.to(dtype), ids, t, lab, lse, T, alpha)


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("up", [1.0, 0.25, 3.0])
def test_reductions_and_upstream_gradients(reduction, up):
    s, ids, t, lab, lse = _case(20, 999, 16, 5, labels=True, tail=True, T=2.0)
    _check(s, ids, t, lab, lse, 2.0, 0.6, reduction, up)


@pytest.mark.parametrize("tail", [False, True])
def test_a_token_in_several_entries(tail):
    s, ids, t, lab, lse = _case(8, 500, 24, 6, labels=True, tail=False, pad=False)
    ids[:, 5] = ids[:, 0]
    ids[:, 9] = ids[:, 0]
    ids[3:, 11] = ids[3:, 2]
    ids[7] = ids[7, 0]  # all entries the same token
    if tail:
        lse = torch.logsumexp(t.double(), 1).float() + 0.5
    for dtype in DTYPES:
        _check(s.to(dtype), ids, t, lab, lse, 1.0, 0.5)


def test_many_entries():
    s, ids, t, _, _ = _case(3, 9000, 4096, 7, pad=False)
    _check(s, ids, t, None, None, 1.0, 1.0)
    ids[1, 100:200] = ids[1, 0:100]
    _check(s, ids, t, None, None, 1.0, 1.0)


@pytest.mark.parametrize("mask", ["inf", "lowest"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_logits(mask, dtype):
    """Tokens masked out of the student's vocabulary, the teacher keeping to the others: by -inf, and by the
    type's lowest value."""
    s, ids, t, lab, _ = _case(10, 700, 12, 8, labels=True)
    s = s.to(dtype)
    off = torch.ones_like(s, dtype=torch.bool)
    off.scatter_(1, ids.clamp(min=0), False)
    off[torch.arange(10, device=DEV), lab.clamp(min=0)] = False
    off[:, ::2] &= True
    off[:, 1::2] = False
    s = torch.where(off, torch.full_like(s, -math.inf if mask == "inf" else torch.finfo(dtype).min), s)
    x = s.clone().requires_grad_(True)
    distillation_loss(x, ids, t, lab, alpha=0.5).backward()
    assert torch.isfinite(x.grad).all() and not x.grad[off].any()
    keep = torch.where(off, torch.full_like(s, -1e4 if dtype != torch.float16 else torch.finfo(dtype).min), s)
    y = keep.clone().requires_grad_(True)
    _check(keep, ids, t, lab, None, 1.0, 0.5, grad_of=y)
    assert torch.equal(x.grad, y.grad)


def test_teacher_entries_of_minus_infinity_and_rows_without_entries():
    s, ids, t, _, _ = _case(9, 300, 8, 9, pad=False)
    t[2, 3:] = -math.inf
    t[4] = -math.inf
    ids[5] = -1
    ids[6, 1:] = -7
    _check(s, ids, t, None, None, 1.5, 1.0)
    lab = torch.arange(9, device=DEV)
    _check(s, ids, t, lab, None, 1.5, 0.5)


def test_ignored_rows_are_not_read():
    s, ids, t, lab, lse = _case(12, 4000, 10, 10, labels=True)
    clean = s.clone().requires_grad_(True)
    a = distillation_loss(clean, ids, t, lab, alpha=0.5)
    a.backward()
    dirty = s.clone()
    dirty[lab == -100] = math.nan
    t = torch.where((lab == -100)[:, None], torch.full_like(t, math.nan), t)
    dirty.requires_grad_(True)
    b = distillation_loss(dirty, ids, t, lab, alpha=0.5)
    b.backward()
    assert torch.equal(a, b) and torch.equal(clean.grad, dirty.grad)


def test_a_nan_reaches_the_loss():
    s, ids, t, _, _ = _case(6, 500, 4, 11, pad=False)
    s[2, 77] = math.nan
    row = distillation_loss(s, ids, t, reduction="none")
    assert bool(torch.isnan(row[2])) and int(torch.isnan(row).sum()) == 1


def test_strides_and_alignment():
    big, ids, t, lab, lse = _case(14, 1037, 9, 12, labels=True, tail=True)
    for s in (big[:, :1001], big[:, 3:1004], big[2:, 1:1002], big[::2, :1001], big.t().contiguous().t()[:, :1001]):
        n = s.shape[0]
        _check(s, ids[:n].clamp(max=1000), t[:n], lab[:n].clamp(max=1000), lse[:n], 1.0, 0.5,
               grad_of=s.detach().requires_grad_(True))
    s = big[:, :1001]
    ref = distillation_loss(s, ids, t)
    wide = torch.full((14, 40), -5, device=DEV)
    wide[:, :9] = ids
    assert torch.equal(distillation_loss(s, wide[:, :9], t), ref)
    assert torch.equal(distillation_loss(s, ids.int(), t), ref)
    assert torch.equal(distillation_loss(s.reshape(2, 7, 1001), ids.view(2, 7, 9), t.view(2, 7, 9)), ref)
    # the cut vocabulary leaves some of the teacher's tokens beyond it
    assert _capi.device_status() == (_capi.FF_DEVICE_BADARG if bool((ids >= 1001).any()) else 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_teacher_logits_of_16_bits(dtype):
    s, ids, t, _, _ = _case(7, 800, 12, 13)
    _check(s, ids, t.to(dtype), None, None, 2.0, 1.0)


def test_indexes_beyond_the_vocabulary_are_reported():
    s, ids, t, lab, _ = _case(6, 200, 5, 14, labels=True, pad=False)
    ids2, lab2 = ids.clone(), lab.clone()
    ids2[2, 3] = 200
    lab2[3] = 4000
    got = distillation_loss(s, ids2, t, lab2, alpha=0.5)
    assert _capi.device_status() == _capi.FF_DEVICE_BADARG
    ids[2, 3], lab[3] = -1, -100
    assert torch.equal(got, distillation_loss(s, ids, t, lab, alpha=0.5))
    assert _capi.device_status() == 0


def test_no_rows_and_no_counted_rows():
    x = torch.zeros(0, 50, device=DEV, requires_grad=True)
    e = torch.zeros(0, 3, device=DEV)
    for red in ("mean", "sum"):
        l = distillation_loss(x, e.long(), e, reduction=red)
        assert float(l.detach()) == 0.0
        l.backward()
    assert distillation_loss(x, e.long(), e, reduction="none").shape == (0,)
    s, ids, t, _, _ = _case(4, 50, 3, 15)
    x = s.requires_grad_(True)
    l = distillation_loss(x, ids, t, torch.full((4,), -100, device=DEV), alpha=0.5)
    l.backward()
    assert float(l) == 0.0 and not x.grad.any()


def test_backward_twice_and_without_gradients():
    s, ids, t, lab, _ = _case(30, 3000, 16, 16, labels=True)
    x = s.requires_grad_(True)
    l = distillation_loss(x, ids, t, lab, alpha=0.5)
    (g1,) = torch.autograd.grad(l, x, retain_graph=True)
    first = g1.clone()
    (g2,) = torch.autograd.grad(l * 2, x, retain_graph=True)
    (g3,) = torch.autograd.grad(l, x)
    assert torch.equal(g1, first) and torch.equal(g3, first)
    torch.testing.assert_close(g2.float(), first.float() * 2, rtol=0, atol=0)  # a power of two: no other rounding
    with torch.no_grad():
        assert torch.equal(distillation_loss(x, ids, t, lab, alpha=0.5), l)


def test_same_result_every_time():
    s, ids, t, lab, lse = _case(64, 32000, 64, 17, labels=True, tail=True, T=2.0)
    x = s.requires_grad_(True)
    ref = None
    for _ in range(4):
        l = distillation_loss(x, ids, t, lab, teacher_lse=lse, temperature=2.0, alpha=0.5)
        (g,) = torch.autograd.grad(l, x)
        if ref is not None:
            assert torch.equal(l, ref[0]) and torch.equal(g, ref[1])
        ref = (l.detach(), g)


def test_gradient_against_differences():
    s, ids, t, lab, lse = _case(3, 60, 6, 18, dtype=torch.float32, labels=True, tail=True, T=2.0)
    lab[:] = torch.tensor([3, 5, 7], device=DEV)
    x = s.clone().requires_grad_(True)
    distillation_loss(x, ids, t, lab, teacher_lse=lse, temperature=2.0, alpha=0.5, reduction="sum").backward()
    f = lambda z: O.losses(z, ids, t, lab, lse, 2.0, 0.5)[0].sum()
    h = 1e-4
    for r, v in ((0, 3), (0, int(ids[0, 0])), (1, 59), (2, int(ids[2, 5])), (2, 7)):
        a, b = s.double(), s.double()
        a, b = a.clone(), b.clone()
        a[r, v] += h
        b[r, v] -= h
        diff = float((f(a) - f(b)) / (2 * h))
        # the third derivative is at most alpha T^2 / T^3 + 1 in size: h^2 / 6 of it; fp32 in the kernel
        assert abs(diff - float(x.grad[r, v])) <= 2 * h * h + 1e-10 / h + 2.0 ** -18 * 4


def test_captured_and_replayed_with_another_upstream():
    s, ids, t, lab, _ = _case(40, 5000, 16, 19, labels=True)
    x = s.clone().requires_grad_(True)
    up = torch.ones((), device=DEV)
    def step():
        l = distillation_loss(x, ids, t, lab, alpha=0.5)
        return l, torch.autograd.grad(l, x, up)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        l, grad = step()
    for k, u in enumerate((1.0, 0.5, 1.0, 2.0, 1.0)):
        with torch.no_grad():
            x.copy_(s * (1 + 0.125 * k))
        up.fill_(u)
        g.replay()
        got = l.clone(), grad.clone()
        want = step()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_backward_alone_captured():
    """Only the backward pass is replayed, with one upstream gradient after another."""
    s, ids, t, lab, _ = _case(40, 5000, 16, 20, labels=True)
    x = s.clone().requires_grad_(True)
    up = torch.ones((), device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    # the leaf's first graph is made on the stream that captures: torch refuses to capture a backward pass
    # while an eager graph of the same leaf on the default stream is alive
    with torch.cuda.stream(side):
        l = distillation_loss(x, ids, t, lab, alpha=0.5)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            grad = torch.autograd.grad(l, x, up)[0]
    for u in (1.0, 3.0, 1.0, 1.0, 0.5):
        up.fill_(u)
        g.replay()
        got = grad.clone()
        y = s.clone().requires_grad_(True)
        (want,) = torch.autograd.grad(distillation_loss(y, ids, t, lab, alpha=0.5), y, up.clone())
        assert torch.equal(got, want)


def test_two_streams_at_once():
    cases = [_case(50, 8000, 16, s, labels=True) for s in (21, 22)]
    f = lambda c: distillation_loss(c[0], c[1], c[2], c[3], alpha=0.5)
    wants = [f(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(5):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(f(cases[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for v in got[k]:
            assert torch.equal(v, wants[k])


def test_decoder_distils_from_a_teacher():
    """The decoder's own path: the teacher's top logits, the student's loss, gradients in every parameter."""
    cfg = DecoderConfig(vocab=512, d_model=128, heads=4, ffn=256, layers=2, max_seq=64)
    teacher, student = build_decoder(cfg, DEV, seed=1), build_decoder(cfg, DEV, seed=2)
    ids = torch.randint(0, cfg.vocab, (2, 65), device=DEV)
    with torch.no_grad():
        tl = teacher(ids[:, :-1]).float()
    top = tl.topk(16, dim=-1)
    loss = student.distill_loss(ids[:, :-1], ids[:, 1:], top.indices, top.values,
                                teacher_lse=torch.logsumexp(tl / 2, -1), temperature=2.0, alpha=0.5)
    with torch.no_grad():
        logits = student(ids[:, :-1]).double().view(-1, cfg.vocab)
    want, counted, scale = O.losses(logits, top.indices.view(-1, 16), top.values.view(-1, 16), ids[:, 1:].reshape(-1),
                                    torch.logsumexp(tl / 2, -1).view(-1), 2.0, 0.5)
    assert abs(float(loss) - float(want.mean())) <= 2.0 ** -19 * (4 * (4 + float(scale.max())) + 16)
    loss.backward()
    for lin in student.bit_modules():
        g = lin.consume_weight_grad()
        assert g is not None and torch.isfinite(g).all() and bool(g.any())
    for p in student.dense_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all()


def test_more_than_2_31_logits():
    """Offsets past 32 bits: the last rows of a long batch against the same rows by themselves."""
    n, V, k = 68000, 32000, 8
    s = torch.empty(n, V, device=DEV, dtype=torch.bfloat16)
    s.normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    ids = torch.randint(0, V, (n, k), device=DEV)
    t = torch.randn(n, k, device=DEV)
    x = s.requires_grad_(True)
    distillation_loss(x, ids, t, reduction="sum").backward()
    y = s.detach()[-5:].clone().requires_grad_(True)
    distillation_loss(y, ids[-5:], t[-5:], reduction="sum").backward()
    # another cut of the row into slices: other sums, the same up to their rounding and the output's
    assert bool(((x.grad[-5:].float() - y.grad.float()).abs() <= 2.0 ** -7 * y.grad.float().abs() + 1e-9).all())
    with torch.no_grad():
        rows = distillation_loss(s, ids, t, reduction="none")
        want = distillation_loss(s[-5:].clone(), ids[-5:], t[-5:], reduction="none")
    assert bool(((rows[-5:] - want).abs() <= 2.0 ** -19 * 32).all())


@pytest.mark.parametrize("T", [1e-2, 1e4])
def test_extreme_temperatures(T):
    s, ids, t, lab, _ = _case(6, 900, 10, 30, labels=True)
    x = s.clone().requires_grad_(True)
    l = distillation_loss(x, ids, t, lab, temperature=T, alpha=0.5)
    s64 = s.double().requires_grad_(True)
    rows, counted, scale = O.losses(s64, ids, t, lab, None, T, 0.5)
    want = rows.sum() / sum(counted)
    want.backward()
    tol = 2.0 ** -19 * float((T * T * (4 + scale) + 16).sum()) / sum(counted)
    assert abs(float(l.detach()) - float(want.detach())) <= tol
    l.backward()
    assert torch.isfinite(x.grad).all()
    # the exponential's argument is rounded to 2^-24 of itself, |s| / T log2 e
    arg = float(s.abs().max()) / T * 1.5
    lim = (2.0 ** -18 + 2.0 ** -23 * arg) * 4 * max(T, 1.0) + 2.0 ** -8 * float(s64.grad.abs().max())
    assert float((x.grad.double() - s64.grad).abs().max()) <= lim


def test_backward_alone_replayed_after_its_gradient_was_changed():
    """What a replayed backward pass returns is its caller's: cleared, scaled or added to, it is formed anew."""
    s, ids, t, lab, _ = _case(40, 5000, 16, 38, labels=True)
    x = s.clone().requires_grad_(True)
    y = s.clone().requires_grad_(True)
    (want,) = torch.autograd.grad(distillation_loss(y, ids, t, lab, alpha=0.5), y)
    up = torch.ones((), device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        l = distillation_loss(x, ids, t, lab, alpha=0.5)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            grad = torch.autograd.grad(l, x, up)[0]
    grad.zero_()  # before the first replay, too
    for change in (lambda: grad.zero_(), lambda: grad.mul_(0.5), lambda: grad.add_(want), lambda: None):
        g.replay()
        assert torch.equal(grad, want)
        change()


def test_forward_and_backward_in_graphs_of_their_own():
    s, ids, t, lab, _ = _case(40, 5000, 16, 39, labels=True)
    x = s.clone().requires_grad_(True)
    up = torch.ones((), device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        distillation_loss(x, ids, t, lab, alpha=0.5).backward()
        x.grad = None
        torch.cuda.synchronize()
        fwd, bwd = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(fwd, stream=side):
            l = distillation_loss(x, ids, t, lab, alpha=0.5)
        with torch.cuda.graph(bwd, stream=side):
            grad = torch.autograd.grad(l, x, up)[0]
    for k in range(3):
        x.data.copy_(s * (1 + 0.25 * k))
        y = x.detach().clone().requires_grad_(True)
        ref = distillation_loss(y, ids, t, lab, alpha=0.5)
        (want,) = torch.autograd.grad(ref, y)
        fwd.replay()
        grad.zero_()
        bwd.replay()
        assert torch.equal(l, ref) and torch.equal(grad, want)


def test_a_replayed_forward_leaves_earlier_gradients_alone():
    """A captured loss whose backward pass runs eagerly, step after step: the gradients of earlier steps are summed."""
    s, ids, t, lab, _ = _case(40, 5000, 16, 40, labels=True)
    x = s.clone().requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            l = distillation_loss(x, ids, t, lab, alpha=0.5)
        wants, gots = [], []
        for k in range(3):
            x.data.copy_(s * (1 + 0.25 * k))
            g.replay()
            gots.append(torch.autograd.grad(l, x, retain_graph=True)[0])
            y = x.detach().clone().requires_grad_(True)
            wants.append(torch.autograd.grad(distillation_loss(y, ids, t, lab, alpha=0.5), y)[0])
        torch.cuda.synchronize()
    for a, b in zip(gots, wants):
        assert torch.equal(a, b)


def test_c_entry_that_is_replayed_forms_its_gradient_anew():
    """``held`` of a replayed ff_distill_grad: equal once, then only after ff_distill_loss has run again."""
    s, ids, t, lab, _ = _case(10, 900, 8, 43, labels=True)
    rows = _capi.distill_rows(s, ids, t, lab, None, 1.0, 0.5, -100)
    up = torch.ones((), device=DEV)
    for _ in range(2):
        _, _, grad, held, counts = _capi.distill_loss(rows, s, "mean", True)
        want = grad.clone()
        for _ in range(3):
            assert torch.equal(_capi.distill_grad(rows, s, "mean", up, counts, grad, held, replayed=True), want)
            assert bool(torch.isnan(held))
            grad.zero_()


# ---------------------------------------------------------------------------
# element by element, each rounding counted
# ---------------------------------------------------------------------------
def _bounds(s, ids, t, lab, lse, T, alpha):
    """Rows' losses and gradients in fp64, which rows count, and what fp32 may be off by: per row for the loss, per
    element for the gradient of the rows' sum.  With u = 2^-24, half a step of 1:
      log p: 1/T, t/T and the difference rounded; without lse also log Z, K/32 + 8 additions of exponentials;
      p: that and 4u for the exponential; sum p: K/32 + 8 additions more; p_rest = 1 - sum p: u more;
      an exponential of q with the argument z (base 2): three roundings in log2(e)/T, one in the multiply-add, one where
      the references of two CTAs differ, 5u |z|, and 4u;
      sums over the row: V/512 + 28 additions (in a thread, over the warps, over the CTAs);
      logarithms: 4u of their values;  the loss: K/256 + 16 additions.
    At T = 2 and 4 the softmax at 1 is a square of exponentials: twice (four times) their errors.  The factor 1.05
    covers the terms of second order."""
    u = 2.0 ** -24
    n, V = s.shape
    K = ids.shape[1]
    x = s.detach().double()  # counted from the row's maximum, so that 64 bits hold the logarithms beside a mask of -1e30
    x = (x - x.amax(1, keepdim=True).clamp(min=-1e300)).requires_grad_(True)
    rows, counted, _ = O.losses(x, ids, t, lab, lse, T, alpha)
    rows.sum().backward()
    rows, grad, x = rows.detach(), x.grad, x.detach()
    zero = torch.zeros((), dtype=torch.float64, device=s.device)
    on = (ids >= 0) & (ids < V) & (t != -math.inf)
    at = torch.where(on, ids, 0).long()
    has = on.any(1, keepdim=True)
    tt = torch.where(on, t.double() / T, zero)
    lz = torch.logsumexp(tt.masked_fill(~on, -math.inf), 1, keepdim=True) if lse is None else lse.double()[:, None]
    lp = torch.where(on, tt - torch.where(has, lz, zero), zero)
    p = torch.where(on, torch.exp(lp), zero)
    d_lp = 4 * u * tt.abs() + 2 * u * lp.abs()
    if lse is None:
        d_lp = d_lp + 6 * u * tt.abs().amax(1, keepdim=True) + (K / 32 + 16) * u
    e_p = d_lp + 4 * u
    psum = p.sum(1, keepdim=True)
    d_ps = (e_p * p).sum(1, keepdim=True) + (K / 32 + 8) * u * psum
    gap = (x - x.amax(1, keepdim=True)).abs() * 1.4427
    z = gap / T
    logq = torch.log_softmax(x / T, 1)
    q = torch.exp(logq)
    e_sum = (V / 512 + 28) * u + 5 * u * torch.where(q > 0, q * z, zero).sum(1, keepdim=True)
    e_q = 5 * u * z + 4 * u + e_sum
    lq = logq.gather(1, at)
    d_lq = e_q.gather(1, at) + 4 * u * (1 + math.log(V))
    live = on & (p > 0)
    size = torch.where(live, p * (lp.abs() + lq.abs()), zero).sum(1)
    d_kd = torch.where(live, p * (e_p * (lp.abs() + lq.abs()) + d_lp + d_lq), zero).sum(1)
    mark = torch.zeros(n, V, dtype=torch.bool, device=s.device)
    mark[torch.arange(n, device=s.device)[:, None].expand_as(at)[on], at[on]] = True
    pv = torch.zeros_like(q).scatter_add_(1, at, p)
    tol = q * torch.where(q > 0, e_q, zero) + torch.zeros_like(q).scatter_add_(1, at, (e_p + 2 * u) * p)
    if lse is not None:
        other = ((~mark).any(1, keepdim=True)) & has
        pr = torch.where(other, (1 - psum).clamp(min=0), zero)
        d_pr = torch.where(other, d_ps + u, zero)
        rest = logq.masked_fill(mark, -math.inf)
        lr = torch.where(other, torch.logsumexp(rest, 1, keepdim=True), zero)
        share = torch.where(other, torch.exp(rest - lr), zero)  # softmax over the tokens outside the entries
        zr = lr.abs() * 1.4427
        log_pr = torch.where(pr > 0, torch.log(pr), zero).abs()
        # x log x + x |log q_rest|: by its slope, or where p_rest may be 0 by its size
        d_rest = torch.where(pr > d_pr, 2 * d_pr * (log_pr + 1 + lr.abs()),
                             2 * d_pr * (torch.log(2 * d_pr + 1e-30).abs() + lr.abs()))
        d_kd = d_kd + (d_rest + pr * (e_sum + 10 * u * zr + 4 * u * (lr.abs() + log_pr + 2)))[:, 0]
        size = size + (pr * (log_pr + lr.abs()))[:, 0]
        zz = torch.where(share > 0, (x - x.masked_fill(mark, -math.inf).amax(1, keepdim=True)).abs() / T * 1.4427, zero)
        # (below a rest of 2^-60 of the row, q itself is left out beside the rest's softmax)
        tol = tol + share * (d_pr + pr * (5 * u * (zz + zr.clamp(max=90)) + 12 * u + e_sum + 2.0 ** -59))
        tol = tol * psum.clamp(min=1) + q * d_ps
    d_row = alpha * T * T * torch.where(has[:, 0], d_kd + (K / 256 + 16) * u * size, zero)
    tol = alpha * T * torch.where(has, tol + 2.0 ** -120, zero)
    if lab is not None:
        y = lab.clamp(min=0)[:, None]
        q1 = torch.softmax(x, 1)
        e_1 = (V / 512 + 28) * u + 20 * u * torch.where(q1 > 0, q1 * gap, zero).sum(1, keepdim=True)
        tol = tol + (1 - alpha) * (torch.where(q1 > 0, q1 * (20 * u * gap + 16 * u + e_1), zero) + 2.0 ** -120
                                   + 4 * u * torch.zeros_like(q).scatter_(1, y, 1.0))
        d_row = d_row + (1 - alpha) * (20 * u * gap.gather(1, y) + e_1 + 4 * u * (1 + math.log(V)))[:, 0]
    ok = torch.tensor(counted, device=s.device)
    d_row = torch.where(ok, 1.05 * d_row + 4 * u * rows.abs(), zero)
    return rows, grad, ok, d_row, torch.where(ok[:, None], 1.05 * tol + 6 * u * grad.abs(), zero), mark


def _check_each(s, ids, t, lab=None, lse=None, T=1.0, alpha=1.0):
    """Row losses and the gradient of their sum against fp64, within ``_bounds`` and the gradient's own rounding.
    Returns how much of the gradient off the entries is larger than its bound."""
    rows, grad, ok, d_row, tol, mark = _bounds(s, ids, t, lab, lse, T, alpha)
    kw = dict(teacher_lse=lse, temperature=T, alpha=alpha)
    got = distillation_loss(s, ids, t, lab, reduction="none", **kw).double()
    assert bool(((got - rows).abs() <= d_row).all()), (got.tolist()[:4], rows.tolist()[:4], d_row.tolist()[:4])
    x = s.detach().clone().requires_grad_(True)
    distillation_loss(x, ids, t, lab, reduction="sum", **kw).backward()
    info = torch.finfo(s.dtype)
    tol = tol * (1 + info.eps) + info.eps / 2 * grad.abs() + info.smallest_normal * info.eps
    off = (x.grad.double() - grad).abs()
    bad = ~(off <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float((off / tol.clamp(min=1e-300)).max()), torch.nonzero(bad)[:4].tolist())
    assert _capi.device_status() == 0
    return float((grad.abs() > tol)[~mark & ok[:, None]].double().mean())


@pytest.mark.parametrize("V", [500, 40000])
@pytest.mark.parametrize("T", [1.0, 2.0])
def test_gradient_of_entries_that_sum_to_more_than_one(V, T):
    """A teacher's log-sum-exp of 16 bits, repeated tokens: sum p lies above 1 by percents, and the gradient is still the
    loss's."""
    for dtype in DTYPES:
        s, ids, t, lab, lse = _case(6, V, 24, 34, labels=True, tail=True, T=T, pad=False)
        s = s.to(dtype)
        low = (torch.logsumexp(t.double() / T, 1) - 0.03).float()
        _check_each(s, ids, t, None, low, T)
        _check_each(s, ids, t, lab, low, T, 0.5)
        _check_each(s, ids, t, None, lse.bfloat16().float(), T)
        ids[:, 5:9] = ids[:, :1]
        _check_each(s, ids, t, lab, low, T, 0.5)
    # against differences, in fp32
    s, ids, t, _, _ = _case(2, 60, 6, 35, dtype=torch.float32, pad=False)
    low = (torch.logsumexp(t.double() / T, 1) - 0.5).float()
    x = s.clone().requires_grad_(True)
    distillation_loss(x, ids, t, teacher_lse=low, temperature=T, reduction="sum").backward()
    f = lambda z: O.losses(z, ids, t, None, low, T, 1.0)[0].sum()
    h = 1e-4
    for r, v in ((0, 3), (0, int(ids[0, 0])), (1, 59), (1, int(ids[1, 5]))):
        a, b = s.double().clone(), s.double().clone()
        a[r, v] += h
        b[r, v] -= h
        # the third derivative is at most sum p T^2 / T^3 in size: h^2 / 6 of it; fp32 in the kernel
        assert abs(float((f(a) - f(b)) / (2 * h)) - float(x.grad[r, v])) <= h * h + 1e-10 / h + 2.0 ** -18 * 4


@pytest.mark.parametrize("T,labels", [(0.01, False), (0.01, True), (0.05, False), (0.7, True)])
def test_rows_cut_over_several_ctas_at_small_temperatures(T, labels):
    """Logits that are large against their spread: what is rounded in M log2(e) / T has to cancel between the CTAs (of
    logits near 10 at T = 0.01 it is up to 2^-14)."""
    g = torch.Generator(device=DEV).manual_seed(37)
    n, V, k = 12, 40000, 16
    base = torch.rand(n, 1, device=DEV, generator=g) * 10 + 5
    s = base + T * torch.rand(n, V, device=DEV, generator=g)
    ids = torch.randint(0, V, (n, k), device=DEV, generator=g)
    t = torch.rand(n, k, device=DEV, generator=g) * T
    lab = torch.randint(0, V, (n,), device=DEV, generator=g) if labels else None
    _check_each(s, ids, t, lab, None, T, 0.5 if labels else 1.0)
    lse = torch.full((n,), math.log(V), device=DEV)
    _check_each(s, ids, t, lab, lse, T, 0.5 if labels else 1.0)


@pytest.mark.parametrize("T", [0.01, 0.7, 1.0, 2.0, 3.0, 4.0, 1000.0])
@pytest.mark.parametrize("mask", [-1e9, -1e10, -1e30, "lowest"])
def test_masks_that_fill_a_whole_slice_or_row(mask, T):
    """A vocabulary whose upper half is masked (one CTA's slice and more hold nothing else), rows of nothing but the mask,
    and rows of large logits of either sign."""
    for dtype in (torch.float32, torch.bfloat16):
        low = torch.finfo(dtype).min if mask == "lowest" else mask
        s, ids, t, lab, _ = _case(5, 32768, 8, 36, labels=True, pad=False)
        ids, lab = ids % 16000, torch.where(lab >= 0, lab % 16000, lab)
        s = s.to(dtype)
        s[:, 16384:] = low
        s[1] = low
        s[2, :16000] += 64 if mask == -1e9 else 0
        _check_each(s, ids, t, None, None, T)
        _check_each(s, ids, t, lab, None, T, 0.5)
        big = s[3:4].clone()
        big[:, 100] = -low  # one logit above all others: a softmax of one token
        _check_each(big, torch.full_like(ids[3:4], 100), t[3:4], torch.full_like(lab[3:4], 100), None, T, 0.5)


@pytest.mark.parametrize("V", [700, 40000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_masked_label_and_a_masked_entry(V, dtype):
    """The type's lowest value at the label, or at a token that the teacher keeps: a large loss, but a finite one."""
    s, ids, t, lab, _ = _case(4, V, 8, 42, labels=True, pad=False, dtype=dtype)
    lab = lab.clamp(min=0)
    one = s.scatter(1, lab[:, None], torch.finfo(dtype).min)
    _check_each(one, ids, t, lab, None, 1.0, 0.5)
    t[:, 0] -= 8  # little of the teacher's mass: the loss stays in range
    two = s.scatter(1, ids[:, :1], torch.finfo(dtype).min)
    _check_each(two, ids, t)
    _check_each(two, ids, t, None, torch.logsumexp(t.double(), 1).float() + 0.1)


@pytest.mark.parametrize("n,V", [(5, 131071), (3, 250007), (6, 2001)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rest_bucket_gradient_of_every_token(n, V, dtype):
    """Of nearly all the tokens outside the entries the gradient is larger than its bound, so none can be missing."""
    for T in (1.0, 2.0, 4.0):
        s, ids, t, lab, lse = _case(n, V, 100, V, dtype=dtype, labels=True, tail=True, T=T, pad=False)
        seen = _check_each(s, ids, t, None, lse, T)
        if dtype == torch.float32:  # (fp16 gradients of a long row are below the type's smallest steps)
            assert seen > 0.95
        _check_each(s, ids, t, lab, lse, T, 0.5)


def _far_rest(n, V, k, seed, T, dtype, gap):
    """A student that is sure of the teacher's tokens: every other logit lies about ``gap`` below them, while
    the teacher leaves a tenth of its mass there."""
    s, ids, t, lab, _ = _case(n, V, k, seed, labels=True, pad=False, dtype=torch.float32)
    s = s.scatter(1, ids, s.gather(1, ids) + gap)
    lse = torch.logsumexp(t.double() / T, 1).float() + 0.1
    return s.to(dtype), ids, t, lab, lse


@pytest.mark.parametrize("n,V", [(6, 700), (3, 40000)])
@pytest.mark.parametrize("T,gap", [(1e-2, 10.0), (0.1, 30.0), (0.7, 100.0), (1.0, 80.0), (1.0, 200.0), (1.0, 1e4), (2.0, 400.0),
                                   (3.0, 1000.0), (4.0, 1000.0)])
def test_rest_bucket_far_below_the_entries(n, V, T, gap):
    for dtype in (torch.float32, torch.bfloat16):
        s, ids, t, lab, lse = _far_rest(n, V, 9, 31, T, dtype, gap)
        _check_each(s, ids, t, None, lse, T)
        for label in (lab, ids[:, 0].contiguous()):  # outside the entries, mostly, and among them
            _check_each(s, ids, t, label, lse, T, 0.5)
        ids = ids.clone()
        ids[:, 4] = ids[:, 1]  # a token in two entries
        _check_each(s, ids, t, lab, lse, T, 0.25)


@pytest.mark.parametrize("V", [700, 40000])
def test_rest_bucket_masked_in_the_student(V):
    """Tokens outside the entries masked by -1e4 or the type's lowest value are still there, by -inf they are not: a rest that
    the teacher keeps costs infinitely much then, and one that is only the rounding of 1 - sum p nothing."""
    s, ids, t, _, _ = _case(4, V, 9, 32, pad=False, dtype=torch.float32)
    exact = torch.logsumexp(t.double(), 1).float()
    out = torch.ones_like(s, dtype=torch.bool).scatter_(1, ids, False)
    _check_each(s.masked_fill(out, -1e4), ids, t, None, exact + 0.1)
    far = s.masked_fill(out, -1e30).requires_grad_(True)  # 64 bits do not hold log R beside 1e30: the R tokens are equal, so
    row = distillation_loss(far, ids, t, teacher_lse=exact + 0.1, reduction="none")  # each gets -p_rest / R
    p = torch.exp(t.double() - (exact + 0.1).double()[:, None])
    pr = 1 - p.sum(1)
    # p_rest within 2^-18 (nine logits below 20, each rounded to 2^-24 of itself, nine exponentials)
    assert bool(((row.double() / (pr * 1e30) - 1).abs() <= 2.0 ** -18 / pr).all())
    row.sum().backward()
    want = (-pr / out.sum(1))[:, None].expand_as(s)
    assert bool(((far.grad - want)[out].abs() <= (2.0 ** -18 / out.sum(1))[:, None].expand_as(s)[out]).all())
    q = torch.softmax(s.gather(1, ids).double(), 1)
    assert bool(((far.grad.gather(1, ids) - (q - p)).abs() <= 2.0 ** -18).all())
    gone = s.masked_fill(out, -math.inf)
    x = gone.clone().requires_grad_(True)
    rows = distillation_loss(x, ids, t, teacher_lse=exact + 0.1, reduction="none")
    assert bool((rows == math.inf).all())
    rows = distillation_loss(x, ids, t, teacher_lse=exact, reduction="none")
    near = distillation_loss(x, ids, t, reduction="none")
    # sum p is 1 to 2^-20: so are the losses, of logits below 20
    assert bool(((rows - near).abs() <= 2.0 ** -20 * 64).all())
    rows.sum().backward()
    assert torch.isfinite(x.grad).all() and not x.grad[out].any()


@pytest.mark.parametrize("off", [-0.05, 0.05, 0.0])
@pytest.mark.parametrize("V", [1, 40, 1000, 4096])
def test_entries_that_cover_the_vocabulary_leave_no_rest(V, off):
    """No token is outside the entries: the bucket is empty whatever 1 - sum p says (a teacher's lse of 16 bits)."""
    s, ids, t, lab, _ = _case(3, V, V, 33, labels=True, pad=False)
    lse = torch.logsumexp(t.double(), 1).float() + off
    _check_each(s, ids, t, None, lse)
    _check_each(s, ids, t, lab, lse, 1.0, 0.5)


@pytest.mark.parametrize("T", [0.01, 0.7, 1.0, 2.0, 4.0])
@pytest.mark.parametrize("mask", [-1e10, "lowest"])
def test_rest_bucket_over_whole_masked_slices(mask, T):
    for dtype in (torch.float32, torch.bfloat16):
        s, ids, t, lab, _ = _case(4, 32768, 8, 44, labels=True, pad=False)
        ids, lab = ids % 16000, torch.where(lab >= 0, lab % 16000, lab)
        s = s.to(dtype)
        s[:, 16384:] = torch.finfo(dtype).min if mask == "lowest" else mask
        lse = torch.logsumexp(t.double() / T, 1).float() + 0.1
        _check_each(s, ids, t, None, lse, T)
        _check_each(s, ids, t, lab, lse, T, 0.5)
        s[1] = s[1, -1]  # nothing but the mask
        _check_each(s, ids, t, None, lse, T)


def test_forward_mode_is_refused_as_by_the_other_layers():
    """There is no forward-mode derivative: a tangent is refused and not lost, with or without ``requires_grad``."""
    from torch.autograd import forward_ad

    s, ids, t, _, _ = _case(3, 50, 4, 41, dtype=torch.float32)
    for x in (s, s.clone().requires_grad_(True)):
        with forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="forward"):
                distillation_loss(forward_ad.make_dual(x, torch.ones_like(x)), ids, t)
            assert torch.equal(distillation_loss(s, ids, t), distillation_loss(s.clone(), ids, t))  # no tangent: as ever


@pytest.mark.parametrize("V,n", [(700, 3000), (9000, 2000), (40000, 900)])
@pytest.mark.parametrize("labels", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_every_kind_one_after_another(V, n, labels, dtype):
    """Ordinary rows, rows whose rest is far below, masked slices, nothing but a mask, no rest, repeated tokens and ignored rows in
    turn on the same CTAs: each as by itself, and the same wherever it stands."""
    T = 2.0
    s, ids, t, lab, _ = _case(8, V, 9, 45, labels=True, pad=False, dtype=torch.float32)
    lse = torch.logsumexp(t.double() / T, 1).float() + 0.1
    s[1].scatter_(0, ids[1], s[1, ids[1]] + 500)  # far rest
    s[2, V // 2:] = -1e10
    s[3] = -1e10
    ids[4, 3:6] = ids[4, 0]
    lab = lab.clamp(min=0)
    lab[5] = -100
    ids[6] = -1
    s[7].scatter_(0, ids[7], s[7, ids[7]] - 500)  # next to nothing on the entries
    s, lab = s.to(dtype), lab if labels else None
    _check_each(s, ids, t, lab, lse, T, 0.5 if labels else 1.0)
    kind = torch.randint(0, 8, (n,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(46))
    kind[:8] = torch.arange(8, device=DEV)
    first = torch.stack([torch.nonzero(kind == k)[0, 0] for k in range(8)])
    lab_n = None if lab is None else lab[kind]
    x = s[kind].requires_grad_(True)
    kw = dict(teacher_lse=lse[kind], temperature=T, alpha=0.5 if labels else 1.0)
    rows = distillation_loss(x, ids[kind], t[kind], lab_n, reduction="none", **kw)
    loss = distillation_loss(x, ids[kind], t[kind], lab_n, reduction="sum", **kw)
    loss.backward()
    assert torch.equal(rows, rows[first][kind]) and torch.equal(x.grad, x.grad[first][kind])
    # each row as in the batch of eight, whose rows may be cut into other slices
    want, grad, ok, d_row, tol, _ = _bounds(s, ids, t, lab, lse, T, 0.5 if labels else 1.0)
    assert bool(((rows[first].double() - want).abs() <= d_row).all())
    info = torch.finfo(dtype)
    tol = tol * (1 + info.eps) + info.eps / 2 * grad.abs() + info.smallest_normal * info.eps
    assert bool(((x.grad[first].double() - grad).abs() <= tol).all())
    assert _capi.device_status() == 0
