"""What the losses refuse, on the host and before any launch."""
from __future__ import annotations

import ctypes

import pytest
import torch


def _logits(**kw):
    from engraft_ngram_amd import _lib
    base = dict(data=256, dtype=1, targets_i32=0, n=4, v=100, row_stride=100, targets=256, temperature=1.0)
    base.update(kw)
    return _lib.EgLogits(*[base[f] for f, _ in _lib.EgLogits._fields_])


def _refusal(fn, *args):
    from engraft_ngram_amd import _lib
    rc = fn(*args)
    return rc, (_lib.load().eg_last_error() or b"").decode()


@pytest.mark.parametrize("needle,bad", [
    ("dtype=7", dict(dtype=7)), ("n=-1", dict(n=-1)), ("v=0", dict(v=0)), ("row_stride=99", dict(row_stride=99)),
    ("temperature=0", dict(temperature=0.0)), ("temperature=nan", dict(temperature=float("nan"))),
    ("temperature=inf", dict(temperature=float("inf"))), ("NULL", dict(data=None)), ("NULL", dict(targets=None)),
    ("aligned", dict(data=257)), ("v=2147483647", dict(v=2 ** 31 - 1, row_stride=2 ** 31)),
])
def test_logits_are_checked(needle, bad):
    from engraft_ngram_amd import _lib
    lib = _lib.load()
    l = _logits(**bad)
    rc, msg = _refusal(lib.eg_token_logprobs, ctypes.byref(l), 256, 256, 1 << 20, None)
    assert rc == _lib.EG_ERR_ARG and needle in msg
    rc, msg = _refusal(lib.eg_logits_grad, ctypes.byref(l), 256, None, 1.0, 256, 1 << 40, None)
    assert rc == _lib.EG_ERR_ARG and needle in msg


def test_losses_are_checked():
    from engraft_ngram_amd import _lib
    lib = _lib.load()
    l = _logits()

    def policy(d=None, stride=0, ws=1 << 20, **kw):
        p = _lib.EgPolicy(256, 256, 256, 256, 3, 0, 2, 0.2, 0.2, 0.1)
        for k, x in kw.items():
            setattr(p, k, x)
        return _refusal(lib.eg_policy_loss, ctypes.byref(l), ctypes.byref(p), 256, 256, 256, d, stride, 1.0, 256, ws, None)

    for needle, args in (("advantages", dict(advantages=None)), ("reduction=3", dict(reduction=3)),
                         ("clip", dict(clip_low=1.5)), ("clip", dict(clip_high=-0.1)),
                         ("n_segments=-1", dict(n_segments=-1)), ("segment_ids", dict(segment_ids=None)),
                         ("d_stride=99", dict(d=512, stride=99)), ("row stride", dict(d=256, stride=128))):
        rc, msg = policy(**args)
        assert rc == _lib.EG_ERR_ARG and needle in msg, msg
    rc, msg = policy(ws=8)
    assert rc == _lib.EG_ERR_WORKSPACE and "needed" in msg
    for needle, p in (("n_pairs=0", _lib.EgPreference(256, 256, 0, 0, 0.1, 0.0)),
                      ("ref_logprobs", _lib.EgPreference(256, None, 1, 0, 0.1, 0.0)),
                      ("segment_ids", _lib.EgPreference(None, 256, 1, 0, 0.1, 0.0)),
                      ("label_smoothing", _lib.EgPreference(256, 256, 1, 0, 0.1, 1.5))):
        rc, msg = _refusal(lib.eg_preference_loss, ctypes.byref(l), ctypes.byref(p), 256, 256, 256, 256, 256, None, 0,
                           1.0, 256, 1 << 20, None)
        assert rc == _lib.EG_ERR_ARG and needle in msg, msg
    assert lib.eg_loss_workspace_size(-1, 5, 0, 0) == -1 and lib.eg_loss_workspace_size(1, 5, 0, 0) > 0


def test_python_arguments_are_checked():
    """Tensors on the host, of other types or shapes never reach the library."""
    from engraft_ngram_amd import losses
    z, t = torch.zeros((3, 5)), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="on the GPU"):
        losses.token_logprobs(z, t)
    with pytest.raises(ValueError, match="logits must be"):
        losses.token_logprobs(z.double(), t)
    with pytest.raises(ValueError, match="logits must be"):
        losses.policy_loss(z[0], t, t.float())
    with pytest.raises(ValueError, match="logits must be"):
        losses.preference_loss(z, t, t, torch.zeros(2))


@pytest.mark.gpu
def test_python_arguments_are_checked_on_the_gpu(cuda):
    from engraft_ngram_amd import losses
    z, t, a = torch.zeros((3, 6), device=cuda), torch.zeros(3, dtype=torch.int64, device=cuda), torch.zeros(3, device=cuda)
    for match, call in (
            ("unit stride", lambda: losses.token_logprobs(z.T.contiguous().T, t)),
            ("targets must be", lambda: losses.token_logprobs(z, t[:2])),
            ("targets must be", lambda: losses.token_logprobs(z, t.cpu())),
            ("int64 or int32", lambda: losses.token_logprobs(z, a)),
            ("temperature", lambda: losses.token_logprobs(z, t, temperature=-1.0)),
            ("row_stride", lambda: losses.token_logprobs(z[:1].expand(3, 6), t)),
            ("advantages", lambda: losses.policy_loss(z, t, a[:1])),
            ("old_logprobs", lambda: losses.policy_loss(z, t, a, t)),
            ("ref_logprobs", lambda: losses.policy_loss(z, t, a, kl_coef=0.1)),
            ("reduction", lambda: losses.policy_loss(z, t, a, reduction="mean")),
            ("segment_ids", lambda: losses.policy_loss(z, t, a, reduction="sequence")),
            ("clip", lambda: losses.policy_loss(z, t, a, clip=(2.0, 0.1))),
            ("out must be", lambda: losses.policy_loss_grad(z, t, a, out=z.half())),
            ("out must be", lambda: losses.policy_loss_grad(z, t, a, out=z[:2])),
            (r"2 \* pairs", lambda: losses.preference_loss(z, t, t, a)),
            ("label_smoothing", lambda: losses.preference_loss(z, t, t, a[:2], label_smoothing=2.0))):
        with pytest.raises(ValueError, match=match):
            call()


def test_overlapping_gradients_are_refused():
    """d_logits in the logits' place, apart, or between their rows; over some of them or another argument never.  Elements of
    bf16; 4 rows of 100 at 0, 250 apart."""
    from engraft_ngram_amd import _lib
    lib = _lib.load()
    base, far = 1 << 30, 1 << 40
    l = _logits(data=base, row_stride=250, targets=far)
    p = _lib.EgPolicy(far + 1000, far + 2000, far + 3000, far + 4000, 3, 0, 2, 0.2, 0.2, 0.1)
    q = _lib.EgPreference(far + 1000, far + 2000, 3, 0, 0.1, 0.0)

    def calls(at, stride):
        at = base + 2 * at
        yield lib.eg_policy_loss, (ctypes.byref(l), ctypes.byref(p), far, far, far, at, stride, 1.0, 256, 0, None)
        yield lib.eg_preference_loss, (ctypes.byref(l), ctypes.byref(q), far, far, far, far, far, at, stride, 1.0, 256, 0, None)

    for at, stride in ((250, 250), (1, 250), (99, 250), (-99, 250), (849, 100), (-300, 100), (0, 249), (-50, 130)):
        for fn, args in calls(at, stride):
            rc, msg = _refusal(fn, *args)
            assert rc == _lib.EG_ERR_ARG and ("overlap the logits" in msg or "row stride" in msg), (at, stride, msg)
        rc, msg = _refusal(lib.eg_logits_grad, ctypes.byref(l), far, None, 1.0, base + 2 * at, stride, None)
        assert rc == _lib.EG_ERR_ARG
    for at, stride in ((0, 250), (100, 250), (-100, 250), (150, 250), (850, 100), (-400, 100)):
        for fn, args in calls(at, stride):  # as far as the workspace, which is too small
            rc, msg = _refusal(fn, *args)
            assert rc == _lib.EG_ERR_WORKSPACE, (at, stride, msg)
    start = (far - base) // 2
    for at, names in ((start + 10, "targets"), (start + 502, "advantages segment_ids"), (start + 1005, "old_logprobs ref_logprobs")):
        for fn, args in calls(at, 100):
            rc, msg = _refusal(fn, *args)
            assert rc == _lib.EG_ERR_ARG and any(f"overlap {x}" in msg for x in names.split()), (at, msg)
