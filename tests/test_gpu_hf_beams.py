"""Beam search over a model with the tiered decode installed: the pool's slots follow the beams."""
import pytest
import torch

from tests import _golden as GD

pytestmark = pytest.mark.gpu


def _model():
    torch.backends.cudnn.allow_tf32 = False
    torch.backends.cuda.matmul.allow_tf32 = False
    # the state term dominates the mixers' outputs, so a state of another beam changes the tokens
    return GD.MG.hf_state_dominant(GD.MG.hf_model(GD.MG.HF["seed"])).cuda().eval()


def _generate(model, ids, K, new):
    out = model.generate(ids, max_new_tokens=new, num_beams=K, do_sample=False, length_penalty=0.0, eos_token_id=None,
                         num_return_sequences=K, return_dict_in_generate=True, output_scores=True)
    return out.sequences.view(ids.shape[0], K, -1), out.sequences_scores.view(ids.shape[0], K)


@pytest.mark.parametrize("install_args", [dict(pb=32, c=4, cold="fp32", corr=1), dict(pb=64, c=3, cold="fp32", corr=1)])
def test_generate_and_beam_search_with_the_exact_readout(install_args):
    """With an fp32 cold slice and the exact readout the installed model is the model: transformers' beam
    search finds the same beams on both, and hf.beam_search finds them too (no end token and no length
    penalty, where both search the same sums)."""
    from nested_ssm_b200 import hf
    ids = torch.randint(0, 90, (2, 9), generator=torch.Generator().manual_seed(3)).cuda()
    K, new = 3, 11
    want, score = _generate(_model(), ids, K, new)
    model = _model()
    hf.install(model, **install_args)
    got, gs = _generate(model, ids, K, new)
    assert torch.equal(got, want)
    torch.testing.assert_close(gs, score, rtol=1e-4, atol=1e-4)
    pools = [m._nssm["pool"] for m in model.modules() if hasattr(m, "_nssm") and isinstance(m._nssm, dict)]
    assert pools and all(int(p.t.max()) == new - 1 for p in pools)
    seqs, scores = hf.beam_search(model, ids, K, new)
    assert torch.equal(seqs, want)
    torch.testing.assert_close(scores, score, rtol=1e-4, atol=1e-4)
    for p in pools:
        p.check_status()


def test_draft_states_follow_the_beams():
    """The hot-only draft: a search with one beam per prompt equals the greedy tokens, and with more
    beams every mixer's draft state of a row is that of a run that decodes the row's sequence alone."""
    from nested_ssm_b200 import hf
    ids = torch.randint(0, 90, (2, 6), generator=torch.Generator().manual_seed(4)).cuda()
    model = _model()
    hf.install(model, pb=32, cold="off")
    greedy = model.generate(ids, max_new_tokens=6, do_sample=False, eos_token_id=None)
    seqs, _ = hf.beam_search(model, ids, 1, 6)
    assert torch.equal(seqs[:, 0], greedy)
    K, new = 3, 6
    seqs, _ = hf.beam_search(model, ids, K, new)
    mixers = [m for m in model.modules() if hasattr(m, "_nssm") and isinstance(m._nssm, dict)]
    # the search leaves the states before its last reorder: one reorder and token less than seqs
    states = [m._nssm["draft"][m._nssm["slots"].long()].clone() for m in mixers]
    rows = seqs[:, :, :-1].reshape(2 * K, -1)
    with torch.no_grad():
        out = model(input_ids=rows[:, :6], use_cache=True)
        for t in range(6, rows.shape[1]):
            out = model(input_ids=rows[:, t:t + 1], past_key_values=out.past_key_values, use_cache=True)
    alone = [m._nssm["draft"][m._nssm["slots"].long()] for m in mixers]
    for i, (a, b) in enumerate(zip(states, alone)):
        a, b = a.view(2, K, *a.shape[1:]), b.view(2, K, *b.shape[1:])
        for p in range(2):
            for r in range(K):      # a final beam's parent is one of the rows
                d = [float((a[p, q] - b[p, r]).abs().max()) for q in range(K)]
                assert min(d) <= 1e-4 * float(b.abs().max()), (i, p, r, d)


def test_beam_search_ends_with_the_end_token():
    from nested_ssm_b200 import hf
    ids = torch.randint(0, 90, (2, 5), generator=torch.Generator().manual_seed(5)).cuda()
    model = _model()
    hf.install(model, pb=32, c=4, cold="fp32", corr=1)
    free, _ = hf.beam_search(model, ids, 4, 8)
    eos = int(free[0, 0, 7])                 # a token that the search chooses
    seqs, scores = hf.beam_search(model, ids, 4, 8, eos_token_id=eos)
    assert bool((scores[:, 1:] <= scores[:, :-1]).all())
    for row in seqs.reshape(-1, seqs.shape[-1])[:, 5:].tolist():
        if eos in row:
            assert set(row[row.index(eos):]) == {eos}
    assert any(eos in r for r in seqs.reshape(-1, seqs.shape[-1])[:, 5:].tolist())
