"""Fine-tuning operators without a GPU: what the Python entry points and the C ABI refuse, before anything is launched."""
import ctypes as C

import numpy as np
import pytest
import torch

from prosim_amd.engine import PsDecisions, PsPolicyTerms, PsPreference, load_library


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__ as ge
    ge.build()
    return load_library()


FAKE = 1 << 20      # (an address that is never followed: every call below ends on the host)


def _d(**kw):
    a = dict(logits=FAKE, rows=4, choices=8, row_stride=8, dtype=0, choice_bits=64, choice=FAKE, mask=None)
    a.update(kw)
    return PsDecisions(*[a[f[0]] for f in PsDecisions._fields_])


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(choices=0), dict(choices=1 << 31), dict(row_stride=7), dict(dtype=3), dict(dtype=-1), dict(choice_bits=16),
                                 dict(logits=None), dict(choice=None), dict(logits=FAKE + 2), dict(dtype=1, logits=FAKE + 1), dict(choice=FAKE + 4)])
def test_c_entries_refuse_bad_decisions(lib, bad):
    d = _d(**bad)
    assert lib.ps_choice_logp(d, FAKE, None, FAKE, 1 << 20, None) == -1
    assert lib.ps_last_error().startswith(b"ps_choice_logp: ")
    assert lib.ps_choice_grad(d, FAKE, FAKE, None, 0, FAKE, None) == -1
    t = PsPolicyTerms(FAKE, FAKE, None, 0.2, 0.2, 0.0, 1.0, 1)
    assert lib.ps_policy_loss(d, t, FAKE, FAKE, FAKE, FAKE, None, None, None, FAKE, 1 << 20, None) == -1
    assert lib.ps_last_error().startswith(b"ps_policy_loss: ")


def test_c_entries_refuse_missing_buffers(lib):
    assert lib.ps_choice_logp(None, FAKE, None, FAKE, 1 << 20, None) == -1
    assert lib.ps_choice_logp(_d(), None, None, FAKE, 1 << 20, None) == -1
    for args in ((None, FAKE, FAKE), (FAKE, None, FAKE), (FAKE, FAKE, None)):
        assert lib.ps_choice_grad(_d(), args[0], args[1], None, 0, args[2], None) == -1
    for d in (_d(), _d(dtype=2)):
        assert lib.ps_choice_grad(d, FAKE, FAKE, None, 0, FAKE + 1, None) == -1 and lib.ps_choice_grad(d, FAKE, FAKE + 4, None, 0, FAKE, None) == -1
    assert lib.ps_choice_logp(_d(), FAKE, FAKE + 4, FAKE, 1 << 20, None) == -1
    assert lib.ps_choice_logp(_d(rows=0, logits=None, choice=None), None, None, None, 0, None) == 0     # (no rows: nothing to do)


@pytest.mark.parametrize("bad", [dict(old_logp=None), dict(advantage=None), dict(clip_low=-0.1), dict(clip_low=1.5), dict(clip_low=float("nan")), dict(clip_high=-1.0),
                                 dict(clip_high=float("nan")), dict(kl_coef=-1.0), dict(kl_coef=float("inf")), dict(kl_coef=0.1), dict(scale=float("nan")),
                                 dict(scale=float("inf"))])
def test_policy_loss_terms(lib, bad):
    a = dict(old_logp=FAKE, advantage=FAKE, ref_logp=None, clip_low=0.2, clip_high=0.2, kl_coef=0.0, scale=1.0, mean=1)
    a.update(bad)
    t = PsPolicyTerms(*[a[f[0]] for f in PsPolicyTerms._fields_])
    assert lib.ps_policy_loss(_d(), t, FAKE, FAKE, FAKE, FAKE, None, None, None, FAKE, 1 << 20, None) == -1
    assert lib.ps_last_error().startswith(b"ps_policy_loss: ")


def test_workspaces_are_checked(lib):
    t = PsPolicyTerms(FAKE, FAKE, None, 0.2, 0.2, 0.0, 1.0, 1)
    need = lib.ps_choice_workspace(_d())
    assert need > 0 and lib.ps_choice_workspace(None) == -1 and lib.ps_choice_workspace(_d(rows=0)) > 0
    assert lib.ps_clip_grads_workspace(1, None, None) == -1 and lib.ps_clip_grads_workspace(0, None, None) == 8
    for ws, size in ((None, need), (FAKE, need - 1), (FAKE + 4, need)):
        assert lib.ps_policy_loss(_d(), t, FAKE, FAKE, FAKE, FAKE, None, None, None, ws, size, None) == -1
        assert lib.ps_choice_logp(_d(), FAKE, None, ws, size, None) == -1
    q = PsPreference(FAKE, None, FAKE, None, None, None, 2, 3, 3, 0.1, 0.0, 1.0, 1)
    need = lib.ps_preference_loss_workspace(2)
    for ws, size in ((None, need), (FAKE, need - 1), (FAKE + 4, need)):
        assert lib.ps_preference_loss(q, FAKE, FAKE, FAKE, ws, size, None) == -1


@pytest.mark.parametrize("bad", [dict(pairs=0), dict(better_steps=-1), dict(better=None), dict(worse=None), dict(beta=float("nan")), dict(label_smoothing=1.1),
                                 dict(label_smoothing=-0.1), dict(scale=float("inf"))])
def test_preference_arguments(lib, bad):
    a = dict(better=FAKE, better_ref=None, worse=FAKE, worse_ref=None, better_mask=None, worse_mask=None, pairs=2, better_steps=3, worse_steps=3, beta=0.1,
             label_smoothing=0.0, scale=1.0, mean=1)
    a.update(bad)
    q = PsPreference(*[a[f[0]] for f in PsPreference._fields_])
    assert lib.ps_preference_loss(q, FAKE, FAKE, FAKE, FAKE, 1 << 20, None) == -1
    assert lib.ps_last_error().startswith(b"ps_preference_loss: ")


def test_clip_tables_are_checked(lib):
    def call(ptr, numel, dtype, max_norm=1.0, eps=1e-6, norm=FAKE, ws=FAKE, size=1 << 20):
        p, n, t = np.array(ptr, np.uint64), np.array(numel, np.int64), np.array(dtype, np.int32)
        return lib.ps_clip_grads(len(ptr), p.ctypes.data, n.ctypes.data, t.ctypes.data, max_norm, eps, norm, ws, size, None)
    assert call([FAKE], [-1], [0]) == -1
    assert call([0], [4], [0]) == -1
    assert call([FAKE], [4], [7]) == -1
    assert call([FAKE + 2], [4], [0]) == -1
    assert call([FAKE + 1], [4], [1]) == -1
    assert call([FAKE], [4], [0], max_norm=-1.0) == -1
    assert call([FAKE], [4], [0], max_norm=float("nan")) == -1
    assert call([FAKE], [4], [0], eps=float("nan")) == -1
    assert call([FAKE], [4], [0], norm=None) == -1
    assert call([FAKE], [4], [0], ws=None) == -1
    assert call([FAKE], [4], [0], size=8) == -1
    n, t = np.array([1, 0, 1 << 33], np.int64), np.array([0, 1, 2], np.int32)
    assert lib.ps_clip_grads_workspace(3, n.ctypes.data, t.ctypes.data) > 8
    assert lib.ps_clip_grads(1, None, None, None, 1.0, 1e-6, FAKE, FAKE, 1 << 20, None) == -1
    assert b"ps_clip_grads" in lib.ps_last_error()


def test_there_is_no_cpu_fallback(lib):
    from prosim_amd import finetune
    x, c = torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError):
        finetune.choice_logp(x, c)
    with pytest.raises(ValueError):
        finetune.policy_loss(x, c, torch.zeros(2), torch.zeros(2))
    with pytest.raises(ValueError):
        finetune.preference_loss(torch.zeros(2, 3), torch.zeros(2, 3))
    with pytest.raises(ValueError):
        finetune.clip_grads_([x], 1.0)
    with pytest.raises(TypeError):
        finetune.choice_logp(x.numpy(), c)
    with pytest.raises(ValueError):
        finetune.clip_grads_([None], 1.0)


def test_dense_and_row_strides(lib):
    """The layouts the operators take without a copy."""
    from prosim_amd import _finetune
    dense, stride = _finetune.dense, _finetune.row_stride
    t = torch.zeros(4, 5, 6)
    assert dense(t) and dense(t.permute(2, 0, 1)) and dense(t[:1]) and dense(torch.zeros(()))
    assert not dense(t[:, :4]) and not dense(t[..., ::2]) and not dense(torch.zeros(1).expand(3))
    pad = torch.zeros(7, 4, 16)
    assert stride(pad) == 16 and stride(pad[..., :9]) == 16
    assert stride(pad[:, 1, :9]) == 64
    assert stride(pad[:, :3, :9]) == -1                  # two strides: copied
    assert stride(pad[:, :1, :9]) == 64                  # the middle dimension has one entry: one stride
    assert stride(torch.zeros(16).expand(5, 16)) == -1   # rows on top of each other: copied
    assert stride(pad.transpose(1, 2)) == -1 and stride(pad[..., ::2]) == -1
    assert stride(pad[..., :1]) == 16 and stride(torch.zeros(9)) == 9
