"""The distillation loss's oracle against torch's losses, and the refusals that need no GPU."""
import ctypes

import pytest
import torch
from torch.nn import functional as F

from firefly_b200 import _capi, distillation_loss
from oracle import distill_oracle as O


def test_oracle_equals_torch_where_torch_has_the_loss():
    g = torch.Generator().manual_seed(0)
    s, z = torch.randn(5, 30, generator=g, dtype=torch.float64), torch.randn(5, 30, generator=g, dtype=torch.float64)
    lab = torch.tensor([3, -100, 7, 0, 29])
    ids = torch.arange(30).expand(5, 30)
    T, alpha = 2.0, 0.3
    kl = F.kl_div(torch.log_softmax(s / T, 1), torch.log_softmax(z / T, 1), log_target=True, reduction="none").sum(1)
    ce = F.cross_entropy(s, lab, reduction="none", ignore_index=-100)
    want = torch.where(lab != -100, alpha * T * T * kl + (1 - alpha) * ce, torch.zeros(5, dtype=torch.float64))
    got, counted, _ = O.losses(s, ids, z, lab, None, T, alpha)
    torch.testing.assert_close(got, want, rtol=1e-12, atol=1e-12)
    assert counted == [True, False, True, True, True]
    # with the teacher's own log-sum-exp, all but two tokens in the entries: the bucket holds the two
    got, _, _ = O.losses(s, ids[:, 2:], z[:, 2:], None, torch.logsumexp(z / T, 1), T, 1.0)
    p, q = torch.softmax(z / T, 1), torch.softmax(s / T, 1)
    rest = p[:, :2].sum(1) * (p[:, :2].sum(1) / q[:, :2].sum(1)).log()
    torch.testing.assert_close(got, T * T * ((p * (p / q).log())[:, 2:].sum(1) + rest), rtol=1e-10, atol=1e-12)


def _args(n=4, V=20, k=3):
    return torch.zeros(n, V), torch.zeros(n, k, dtype=torch.int64), torch.zeros(n, k)


def test_refusals():
    s, ids, t = _args()
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        distillation_loss(s, ids, t)
    for bad in ((s.int(), ids, t), (s.double(), ids, t), (s, ids.float(), t), (s, ids[:3], t), (s, ids, t[:, :2]),
                (s, ids[:, :0], t[:, :0]), (s, ids, t.double()), (s, ids.to(torch.int16), t), (torch.zeros(()), ids, t)):
        with pytest.raises(ValueError):
            distillation_loss(*bad)
    for kw in (dict(labels=torch.zeros(3, dtype=torch.int64)), dict(labels=torch.zeros(4)), dict(teacher_lse=torch.zeros(5)),
               dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("inf")), dict(temperature=float("nan")),
               dict(alpha=1.5), dict(alpha=-0.1), dict(alpha=float("nan")), dict(reduction="batchmean")):
        with pytest.raises(ValueError):
            distillation_loss(s, ids, t, **kw)
    with pytest.raises(ValueError, match="no gradient"):
        distillation_loss(s, ids, t.requires_grad_(True))


def _rows(**kw):
    f = dict(logits=4096, ids=4096, teacher_logits=4096, labels=0, teacher_lse=0, rows=4, vocab=100, top=8, ld_logits=100,
             ld_ids=8, ld_teacher=8, ignore_index=-100, dtype=1, teacher_dtype=0, ids_64=1, labels_64=0, temperature=1.0,
             alpha=1.0)
    f.update(kw)
    return ctypes.byref(_capi.DistillRows(**f))


def test_c_entries_refuse_before_any_launch():
    lib, bad, uns = _capi.lib(), _capi.FF_ERR_INVALID_ARG, _capi.FF_ERR_UNSUPPORTED
    p, n = ctypes.c_void_p(4096), None
    for kw, rc in ((dict(rows=-1), bad), (dict(vocab=0), bad), (dict(top=0), bad), (dict(top=4097, ld_ids=4097, ld_teacher=4097), uns),
                   (dict(ld_logits=99), bad), (dict(ld_ids=7), bad), (dict(ld_teacher=7), bad), (dict(dtype=3), bad),
                   (dict(teacher_dtype=-1), bad), (dict(temperature=0.0), bad), (dict(alpha=2.0), bad), (dict(logits=0), bad),
                   (dict(logits=4097), bad), (dict(rows=1 << 31), uns), (dict(vocab=1 << 30, ld_logits=1 << 30), uns)):
        assert lib.ff_distill_loss(_rows(**kw), 0, p, n, n, 0, n, n, n) == rc, kw
        assert lib.ff_distill_grad(_rows(**kw), 0, p, n, 0, n, p, 1 << 30, n) == rc, kw
    assert lib.ff_distill_loss(_rows(), 3, p, p, n, 0, n, p, n) == bad
    assert lib.ff_distill_loss(_rows(), 1, p, n, n, 0, n, p, n) == bad        # no scalar
    assert lib.ff_distill_loss(_rows(), 1, p, p, n, 0, n, n, n) == bad        # no counts
    assert lib.ff_distill_loss(_rows(), 0, p, n, p, 100, n, n, n) == bad      # a gradient without a reduction
    assert lib.ff_distill_loss(_rows(), 2, p, p, p, 99, n, n, n) == bad
    assert lib.ff_distill_loss(_rows(), 0, n, n, n, 0, n, n, n) == bad
    assert lib.ff_distill_grad(_rows(), 0, p, p, 0, n, p, 100, n) == bad      # held needs a scalar upstream
    assert lib.ff_distill_grad(_rows(), 1, p, n, 0, n, p, 100, n) == bad
    assert lib.ff_distill_grad(_rows(rows=0), 0, n, n, 0, n, n, 100, n) == _capi.FF_OK


def test_a_vocabulary_that_does_not_fit_is_refused():
    """Eight CTAs hold up to 8 x 227 KB of a row: a longer one is refused on the host."""
    lib, p, n = _capi.lib(), ctypes.c_void_p(4096), None
    assert lib.ff_distill_loss(_rows(vocab=1000000, ld_logits=1000000), 0, p, n, n, 0, n, n, n) == _capi.FF_ERR_UNSUPPORTED
    assert b"does not fit" in lib.ff_last_error()


def test_pointers_that_are_not_aligned_to_their_elements_are_refused():
    lib, bad = _capi.lib(), _capi.FF_ERR_INVALID_ARG
    p, n, odd = ctypes.c_void_p(4096), None, ctypes.c_void_p(4097)
    for kw in (dict(logits=4098, dtype=0), dict(ids=4100), dict(ids=4098, ids_64=0), dict(teacher_logits=4098),
               dict(teacher_logits=4097, teacher_dtype=1), dict(labels=4098), dict(labels=4100, labels_64=1), dict(teacher_lse=4098)):
        assert lib.ff_distill_loss(_rows(**kw), 0, p, n, n, 0, n, n, n) == bad, kw
        assert lib.ff_distill_grad(_rows(**kw), 0, p, n, 0, n, p, 100, n) == bad, kw
    assert lib.ff_distill_loss(_rows(), 0, odd, n, n, 0, n, n, n) == bad
    assert lib.ff_distill_loss(_rows(), 1, p, odd, n, 0, n, p, n) == bad
    assert lib.ff_distill_loss(_rows(), 1, p, p, odd, 100, p, p, n) == bad
    assert lib.ff_distill_loss(_rows(), 1, p, p, p, 100, odd, p, n) == bad
    assert lib.ff_distill_loss(_rows(), 1, p, p, n, 0, n, odd, n) == bad
    assert lib.ff_distill_grad(_rows(), 1, odd, n, 0, p, p, 100, n) == bad
    assert lib.ff_distill_grad(_rows(), 1, p, odd, 0, p, p, 100, n) == bad
    assert lib.ff_distill_grad(_rows(), 1, p, n, 0, odd, p, 100, n) == bad
    assert lib.ff_distill_grad(_rows(), 1, p, n, 0, p, odd, 100, n) == bad
