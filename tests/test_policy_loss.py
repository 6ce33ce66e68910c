"""What `policy_loss` and `token_log_probs` refuse, before anything is launched (no GPU needed)."""
import pytest
import torch

from paccmann_polymer_amd import _C
from paccmann_polymer_amd.policy_loss import policy_loss, token_log_probs

R, V = 5, 7


def good(**change):
    a = dict(logits=torch.zeros(R, V), targets=torch.ones(R, dtype=torch.int64), old_log_probs=torch.zeros(R), advantages=torch.zeros(R))
    a.update(change)
    return a


@pytest.mark.parametrize('change,error', [
    (dict(logits=torch.zeros(R, V, 1)), ValueError),
    (dict(logits=torch.zeros(R, 0)), ValueError),
    (dict(logits=torch.zeros(R, V, dtype=torch.float64)), TypeError),
    (dict(logits=torch.zeros(R, V, dtype=torch.float16)), TypeError),
    (dict(targets=torch.ones(R + 1, dtype=torch.int64)), ValueError),
    (dict(targets=torch.ones(R, dtype=torch.int32)), TypeError),
    (dict(old_log_probs=torch.zeros(R, 1)), ValueError),
    (dict(old_log_probs=torch.zeros(R, dtype=torch.float64)), TypeError),
    (dict(advantages=torch.zeros(1)), ValueError),
    (dict(ref_log_probs=torch.zeros(R + 1)), ValueError),
    (dict(kl_coef=0.1), ValueError),
    (dict(kl_coef=float('nan'), ref_log_probs=torch.zeros(R)), ValueError),
    (dict(clip_low=1.5), ValueError),
    (dict(clip_low=-0.1), ValueError),
    (dict(clip_high=-0.1), ValueError),
    (dict(clip_high=float('inf')), ValueError),
    (dict(temperature=0.0), ValueError),
    (dict(temperature=float('nan')), ValueError),
    (dict(temperature=1e-39), ValueError),
    (dict(temperature=float('inf')), ValueError),
    (dict(), _C.PPKError),                                 # all in order, but on the CPU: there is no fallback
])
def test_policy_loss_refuses(change, error):
    with pytest.raises(error):
        policy_loss(**good(**change))


@pytest.mark.parametrize('logits,targets,temperature,error', [
    (torch.zeros(R), torch.ones(R, dtype=torch.int64), 1.0, ValueError),
    (torch.zeros(R, V), torch.ones(R), 1.0, TypeError),
    (torch.zeros(R, V), torch.ones(R - 1, dtype=torch.int64), 1.0, ValueError),
    (torch.zeros(R, V, dtype=torch.int32), torch.ones(R, dtype=torch.int64), 1.0, TypeError),
    (torch.zeros(R, V), torch.ones(R, dtype=torch.int64), -1.0, ValueError),
    (torch.zeros(R, V), torch.ones(R, dtype=torch.int64), 1.0, _C.PPKError),
])
def test_token_log_probs_refuses(logits, targets, temperature, error):
    with pytest.raises(error):
        token_log_probs(logits, targets, temperature=temperature)


@pytest.mark.parametrize('call,code', [
    (lambda L: L.ppk_token_logp_fwd(1, None, 4, None, 1, 4, 0, 1.0, None, None, None), -4),                                  # fp64 logits
    (lambda L: L.ppk_token_logp_fwd(0, None, 4, None, 1, 4, 0, 1.0, None, None, None), -6),
    (lambda L: L.ppk_token_logp_fwd(0, None, 3, None, 1, 4, 0, 1.0, None, None, None), -1),
    (lambda L: L.ppk_token_logp_fwd(0, None, 4, None, -1, 4, 0, 1.0, None, None, None), -1),
    (lambda L: L.ppk_token_logp_fwd(0, None, 4, None, 0, 4, 0, 1.0, None, None, None), 0),                                   # no rows: nothing to do
    (lambda L: L.ppk_token_logp_bwd(0, None, 4, None, 1, 4, 0, 0.0, None, None, None, 4, None), -1),
    (lambda L: L.ppk_policy_loss(0, None, 4, None, 0, 4, 0, 1.0, None, None, None, 0.2, 0.2, 0.0, None, None, None, 4, None, 0, None), -6),
    (lambda L: L.ppk_policy_loss(0, 16, 4, 16, 1, 4, 0, 1.0, 16, 16, None, 0.2, 0.2, 0.5, 16, 16, None, 4, 256, 1 << 20, None), -6),
    (lambda L: L.ppk_policy_loss(0, 16, 4, 16, 1, 4, 0, 1.0, 16, 16, None, 0.2, 0.2, 0.0, 16, 16, None, 4, 256, 8, None), -3),  # a workspace too small
    (lambda L: L.ppk_policy_loss(0, 16, 4, 16, 1, 4, 0, 1.0, 16, 16, None, 2.0, 0.2, 0.0, 16, 16, None, 4, 256, 1 << 20, None), -1),
    (lambda L: L.ppk_policy_loss(0, 18, 4, 16, 1, 4, 0, 1.0, 16, 16, None, 0.2, 0.2, 0.0, 16, 16, None, 4, 256, 1 << 20, None), -2),
    (lambda L: L.ppk_scale_unless_one(3, None, 1, None, None), -4),
    (lambda L: L.ppk_scale_unless_one(0, None, 1, None, None), -6),
])
def test_c_entries_return_codes(call, code):
    assert call(_C.lib) == code
