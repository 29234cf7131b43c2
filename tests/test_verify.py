"""verify_tokens on the CPU: its meaning (KILN_HIP_INTERPRET=1: the library's
CPU meaning) against its definition, that the tokens which come out are
distributed as the target's, and refusals. Results are whole numbers, compared
for equality: both sides sum in 64 bits, and a random number falls between two
orders of summation with a probability below 10^-10."""

import math

import pytest
import torch

import kiln
import packed_reference as ref


@pytest.fixture()
def interpreting(monkeypatch):
    monkeypatch.setenv("KILN_HIP_INTERPRET", "1")


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def check(p):
    got = kiln.verify_tokens(**p)
    for a, b in zip(got, ref.verify(**p)):
        assert a.dtype == torch.int32 and a.tolist() == b
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tree", [True, False], ids=["tree", "chain"])
@pytest.mark.parametrize("probs", [True, False], ids=["probs", "sampled"])
def test_meaning(interpreting, dtype, tree, probs):
    kept = 0
    for n, vocab in ((1, 5), (2, 1), (7, 33), (40, 300)):
        p = ref.drafted(gen(n), 6, n, vocab, dtype, tree, probs)
        kept += int(check(p)[1].sum())
        check(dict(p, tokens=p["tokens"].to(torch.int32), uniforms=p["uniforms"].double()))
    assert kept > 4 * 6       # (some tokens are kept)


def test_unused_and_odd_tokens(interpreting):
    for probs in (True, False):
        p = ref.drafted(gen(3), 5, 6, 20, probs=probs)
        p["parents"] = torch.tensor([[-2, 0, 0, 1, 2, 3], [-1, -1, -1, 0, 1, 2], [-1, 1, 5, 0, -7, 3], [0, 0, 0, 0, 0, 0], [-1, 0, 0, 0, 0, 0]],
                                    dtype=torch.int32)
        p["tokens"][4] = torch.tensor([0, -1, 20, 2 ** 40, 3, 3])
        rows, counts, after = check(p)
        assert counts[0] == 0 and after[0] == -1 and rows[0].tolist() == [-1] * 6 and counts[3] == 0


def test_odd_probabilities(interpreting):
    for probs in (True, False):
        p = ref.drafted(gen(4), 7, 4, 30, probs=probs, tree=False)
        p["target"][0] = 0.0
        p["target"][1, :, ::2] = math.nan
        p["target"][2, :, 3] = math.inf
        p["target"][3] *= -1.0
        p["target"][4] = p["target"][4] * 0 + torch.eye(30)[7]
        p["uniforms"][5] = torch.tensor([1.0, 0.0, math.nan, -3.0])
        p["uniforms"][6] = 1.0 - 2.0 ** -24
        if probs:
            p["draft"][1, :, 5] = math.nan
            p["draft"][6] = p["target"][6]       # nothing is left after a refusal, if one came
            p["uniforms"][6] = 1.0
        check(p)


def odd_drafts(p):
    """The operands with probabilities of the draft that are negative, and with 0 in their places."""
    draft = p["draft"].clone()
    draft[:, :, ::3] *= -1.0
    draft[0, 0, int(p["tokens"][0, 1])] = -0.5          # asked first, where the target has nothing
    target = p["target"].clone()
    target[0, 0, int(p["tokens"][0, 1])] = 0.0
    p = dict(p, target=target)
    return dict(p, draft=draft), dict(p, draft=torch.where(draft < 0, 0.0, draft))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_draft_probabilities_that_count_as_nothing(interpreting, dtype):
    for seed in range(5):
        p = ref.drafted(gen(seed), 6, 9, 40, dtype, noise=2.0)
        p["uniforms"][0, 1] = 0.9
        odd, want = odd_drafts(p)
        rows, counts, _ = check(want)
        assert [t.tolist() for t in kiln.verify_tokens(**odd)] == [t.tolist() for t in kiln.verify_tokens(**want)]
        assert 1 not in rows[0].tolist() or int(p["parents"][0, 1]) != 0


@pytest.mark.parametrize("probs", [True, False], ids=["probs", "sampled"])
def test_distribution(interpreting, probs):
    # the token behind the root, kept or drawn, is distributed as the target's row: 40000 trials of a root with three
    # children, whatever the draft. 6 standard deviations of a count.
    trials, vocab, g = 40000, 6, gen(5)
    target = torch.tensor([0.3, 0.05, 0.25, 0.2, 0.0, 0.2])
    draft = torch.tensor([0.1, 0.4, 0.1, 0.1, 0.2, 0.1])
    tokens = torch.cat([torch.zeros(trials, 1, dtype=torch.long), torch.multinomial(draft, 3 * trials, True, generator=g).view(trials, 3)], 1)
    parents = torch.tensor([-1, 0, 0, 0], dtype=torch.int32).expand(trials, 4)
    rows, counts, after = kiln.verify_tokens(tokens[:, :4], target.expand(trials, 4, vocab), torch.rand(trials, 4, generator=g, dtype=torch.float64),
                                             parents, draft=draft.expand(trials, 4, vocab) if probs else None) if trials <= 65535 else None
    first = torch.where(counts > 1, tokens.gather(1, rows[:, 1:2].clamp(min=0).long())[:, 0], after.long())
    seen = torch.bincount(first, minlength=vocab).double()
    assert bool(((seen - trials * target).abs() <= 6 * (trials * target * (1 - target)).sqrt()).all()), seen


def test_rows_that_do_not_sum_to_one(interpreting):
    # a target of (0.6, 1.4): without the draft, token 0 for random numbers below 0.3; with it (0.5, 0.5) the two are
    # compared as they are, so both tokens are kept
    n = 100
    target, draft = torch.tensor([0.6, 1.4]).expand(n, 2, 2), torch.tensor([0.5, 0.5]).expand(n, 2, 2)
    u = ((torch.arange(n) + 0.5) / n).double()[:, None].expand(n, 2)
    tokens = torch.tensor([[0, 0]]).expand(n, 2)
    _, counts, after = kiln.verify_tokens(tokens, target, u)
    assert counts.tolist() == [2] * 30 + [1] * 70 and after.tolist() == [0] * 30 + [1] * 70
    for token in (0, 1):
        assert kiln.verify_tokens(tokens + token, target, u, draft=draft)[1].tolist() == [2] * n


def test_strides(interpreting):
    p = ref.drafted(gen(6), 3, 5, 17)
    want = [t.tolist() for t in kiln.verify_tokens(**p)]
    q = dict(p, tokens=p["tokens"].t().contiguous().t(), target=p["target"].transpose(1, 2).contiguous().transpose(1, 2),
             uniforms=torch.stack([p["uniforms"]] * 2, -1)[..., 0], draft=torch.cat([p["draft"]] * 2, 1)[:, :5],
             parents=p["parents"].t().contiguous().t())
    assert [t.tolist() for t in kiln.verify_tokens(**q)] == want
    same = p["target"][:, :1].expand(3, 5, 17)     # one row for all tokens
    assert [t.tolist() for t in kiln.verify_tokens(**dict(p, target=same))] == list(ref.verify(**dict(p, target=same)))


def test_results_of_their_own(interpreting):
    # a result that is kept or saved keeps no other, and no workspace
    results = kiln.verify_tokens(**ref.drafted(gen(8), 3, 5, 17))
    assert [t.untyped_storage().nbytes() for t in results] == [4 * 15, 4 * 3, 4 * 3]
    assert all(t._base is None and t.is_contiguous() and t.storage_offset() == 0 for t in results)


def test_refusals(interpreting):
    p = ref.drafted(gen(), 2, 3, 7)
    for change, error in (
            (dict(tokens=p["tokens"].float()), TypeError), (dict(tokens=p["tokens"][0]), ValueError), (dict(tokens=None), TypeError),
            (dict(target=p["target"].double()), TypeError), (dict(target=p["target"][:, :2]), ValueError), (dict(target=p["target"][..., :0]), ValueError),
            (dict(uniforms=p["uniforms"].half()), TypeError), (dict(uniforms=p["uniforms"][:1]), ValueError),
            (dict(parents=p["parents"].long()), TypeError), (dict(parents=p["parents"][:, :1]), ValueError),
            (dict(draft=p["draft"].bfloat16()), TypeError), (dict(draft=p["draft"][..., :6]), ValueError),
            (dict(target=p["target"].clone().requires_grad_()), NotImplementedError)):
        with pytest.raises(error):
            kiln.verify_tokens(**dict(p, **change))
    with pytest.raises(ValueError):
        kiln.verify_tokens(**{k: None if t is None else t[:, :0] for k, t in p.items()})
    with pytest.raises(NotImplementedError):
        kiln.verify_tokens(**ref.drafted(gen(), 1, 257, 3))
    with pytest.raises(NotImplementedError):     # (a view: no such memory)
        kiln.verify_tokens(p["tokens"], torch.zeros(1).expand(2, 3, 2 ** 24 + 1), p["uniforms"])
    rows, counts, after = kiln.verify_tokens(**{k: t[:0] for k, t in p.items()})
    assert rows.shape == (0, 3) and counts.shape == after.shape == (0,)


def test_transforms_are_refused(interpreting):
    from torch.autograd import forward_ad

    p = ref.drafted(gen(), 2, 3, 7)
    kiln.verify_tokens(**p)
    for name, t in p.items():
        with pytest.raises(RuntimeError):
            torch.vmap(lambda t: kiln.verify_tokens(**dict(p, **{name: t})))(torch.stack([t] * 2))
    for name in ("target", "uniforms", "draft"):
        with pytest.raises(NotImplementedError):
            torch.func.jvp(lambda t: kiln.verify_tokens(**dict(p, **{name: t}))[0].float(), (p[name],), (p[name],))
        with forward_ad.dual_level(), pytest.raises(NotImplementedError):
            kiln.verify_tokens(**dict(p, **{name: forward_ad.make_dual(p[name], p[name])}))


def test_no_cpu_path():
    with pytest.raises(NotImplementedError):
        kiln.verify_tokens(**ref.drafted(gen(), 2, 3, 7))
