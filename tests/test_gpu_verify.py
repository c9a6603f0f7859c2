"""Verification of drafted tokens against its definition in 64 bits."""
import numpy as np
import pytest
import torch

from draftutil import DTYPES, random_parents, verdict

pytestmark = pytest.mark.gpu


def dev(a, dtype=np.int32):
    return torch.from_numpy(np.ascontiguousarray(a, dtype)).cuda()


def run(target, tokens, uniforms, indptr, parents=None, draft=None):
    from deserve_amd.draft_ops import verify_drafts

    got = verify_drafts(target, dev(tokens), dev(uniforms, np.float32), dev(indptr),
                        parents=None if parents is None else dev(parents), draft_probs=draft)
    want = verdict(target.double().cpu().numpy(), tokens, np.asarray(uniforms, np.float32), indptr, parents,
                   None if draft is None else draft.double().cpu().numpy())
    for name, w in zip(("counts", "path", "tokens"), want):
        g = getattr(got, name).cpu().numpy()
        assert np.array_equal(g, w), (name, np.flatnonzero(g != w)[:5], g[g != w][:5], w[g != w][:5])
    return got


def make(seed, rows, vocab, dtype, spread=3.0):
    gen = torch.Generator("cuda").manual_seed(seed)
    total = sum(rows)
    logits = spread * torch.randn((total, vocab), generator=gen, device="cuda")
    target = torch.softmax(logits, 1).to(DTYPES[dtype])
    draft = torch.softmax(logits + 0.5 * torch.randn((total, vocab), generator=gen, device="cuda"), 1).to(DTYPES[dtype])
    indptr = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    uniforms = torch.rand((total,), generator=gen, device="cuda").cpu().numpy()
    return target, draft, indptr, uniforms


def sampled(draft, indptr, parents, seed):
    """Every row's token from the draft's row at its parent."""
    up = []
    for b in range(len(indptr) - 1):
        for i in range(indptr[b + 1] - indptr[b]):
            up.append(int(indptr[b]) + max(0, i - 1 if parents is None else int(parents[indptr[b] + i])))
    gen = torch.Generator("cuda").manual_seed(seed)
    return torch.multinomial(draft.float()[torch.tensor(up, device="cuda")] + 1e-30, 1, generator=gen)[:, 0].cpu().numpy()


@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 4095, 4096, 4097, 32003, 128000])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "f16"])
def test_chains_and_trees(vocab, dtype):
    rows = [1, 5, 0, 64, 2, 7, 0, 33] if vocab < 100000 else [5, 1, 9]
    for seed in range(3):
        target, draft, indptr, uniforms = make(seed, rows, vocab, dtype)
        chain = sampled(draft, indptr, None, seed)
        run(target, chain, uniforms, indptr, draft=draft)
        run(target, chain, uniforms, indptr)
        rng = np.random.default_rng(seed)
        parents = np.concatenate([random_parents(rng, n, 64 if seed == 2 else 4) for n in rows])
        run(target, sampled(target, indptr, parents, seed), uniforms, indptr, parents)


def test_rows_apart():
    rows = [5, 3, 8]
    target, draft, indptr, uniforms = make(1, rows, 1001, "bf16")
    wide = torch.zeros((16, 2, 1007), dtype=torch.bfloat16, device="cuda")
    wide[:, 0, 3:1004], wide[:, 1, 3:1004] = target, draft
    tokens = sampled(draft, indptr, None, 4)
    run(wide[:, 0, 3:1004], tokens, uniforms, indptr, draft=wide[:, 1, 3:1004])


def test_one_hot_rows_verify_greedily():
    rng = np.random.default_rng(0)
    rows, vocab = [9] * 40, 500
    best = rng.integers(0, vocab, sum(rows))
    target = torch.nn.functional.one_hot(torch.from_numpy(best), vocab).float().cuda()
    indptr = np.arange(0, 361, 9, dtype=np.int32)
    parents = np.concatenate([random_parents(rng, 9) for _ in rows])
    tokens = rng.integers(0, vocab, 360)
    right = rng.random(360) < 0.6
    up = np.repeat(indptr[:-1], 9) + np.maximum(parents, 0)
    tokens[right] = best[up][right]
    got = run(target, tokens, rng.random(360), indptr, parents)
    given, counts = got.tokens.cpu().numpy(), got.counts.cpu().numpy()
    for b in range(40):       # the last token is the best one behind the walk
        last = indptr[b] + int(got.path[indptr[b] + counts[b] - 1])
        assert given[indptr[b] + counts[b] - 1] == best[last]


def test_distributions_without_mass_and_values_that_are_none():
    rows, vocab = [3, 3, 3, 3, 3, 3, 1], 700
    target, draft, indptr, uniforms = make(2, rows, vocab, "fp32")
    tokens = sampled(draft, indptr, None, 3)
    uniforms[:] = 0.999
    draft[0:3] = target[0:3]                                     # p = q: nothing is left of p - q
    uniforms[1] = 1.0                                            # and yet refused
    target[3:6] = 0                                              # no mass at all
    target[6, :] = 0
    target[6, tokens[7]] = 1e-3                                  # all mass on the proposed token
    target[9, ::3], target[9, 1], target[9, 2] = float("nan"), float("inf"), -1.0
    tokens[13], tokens[16] = -1, vocab                           # no such tokens
    run(target, tokens, uniforms, indptr, draft=draft)
    run(target, tokens, uniforms, indptr)
    uniforms[[0, 3, 6, 9, 12, 15, 18]] = 0
    run(target, tokens, uniforms, indptr, draft=draft)
    uniforms[[0, 3, 6, 9, 12, 15, 18]] = [1.0, 2.0, np.nan, -1.0, np.inf, 0.5, 1.0]
    run(target, tokens, uniforms, indptr)


def test_the_same_token_among_siblings():
    vocab = 50
    target, _, indptr, _ = make(3, [6] * 200, vocab, "fp32", spread=1.0)
    rng = np.random.default_rng(1)
    parents = np.tile(np.array([-1, 0, 0, 0, 0, 0], np.int32), 200)
    tokens = rng.integers(0, 2, 1200)                            # two tokens for five children
    got = run(target, tokens, rng.random(1200), indptr, parents)
    assert set(got.counts.tolist()) == {1, 2}


def test_given_tokens_are_distributed_as_the_targets():
    """20 000 requests of three rows over 5 tokens: the first token given follows the target's row 0 whatever the
    drafts.  A count of n draws with probability p is off by less than 5 sqrt(n p (1 - p)) but once in 1e6."""
    n, vocab = 20000, 5
    gen = torch.Generator("cuda").manual_seed(5)
    p = torch.tensor([0.05, 0.1, 0.4, 0.15, 0.3], device="cuda")
    q = torch.tensor([0.3, 0.05, 0.2, 0.4, 0.05], device="cuda")
    target, draft = p.repeat(3 * n, 1), q.repeat(3 * n, 1)
    indptr = torch.arange(0, 3 * n + 1, 3, dtype=torch.int32, device="cuda")
    uniforms = torch.rand((3 * n,), generator=gen, device="cuda")
    tokens = torch.multinomial(draft, 1, generator=gen)[:, 0].int()
    from deserve_amd.draft_ops import verify_drafts

    tree = torch.tensor([-1, 0, 0], dtype=torch.int32, device="cuda").repeat(n)
    for kw in (dict(draft_probs=draft), dict(), dict(parents=tree)):
        first = verify_drafts(target, tokens, uniforms, indptr, **kw).tokens.view(n, 3)[:, 0]
        count = torch.bincount(first, minlength=vocab).double()
        assert ((count - n * p).abs() < 5 * (n * p * (1 - p)).sqrt()).all(), (kw.keys(), count / n)


def test_more_rows_than_a_tree_has_and_rows_behind_the_last():
    target, draft, _, uniforms = make(4, [80], 300, "f16")
    tokens = sampled(draft, np.array([0, 80]), None, 1)
    run(target, tokens, uniforms, np.array([0, 65, 70, 70]))
    run(target, tokens, uniforms, np.array([0, 0, 64]), draft=draft)
    run(target[:0], tokens[:0], uniforms[:0], np.array([0, 0, 0]))
    run(target, tokens, uniforms, np.array([0]))


@pytest.mark.parametrize("vocab", [300, 4097, 128000])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "f16"])
@pytest.mark.parametrize("chain", [False, True])
def test_rows_without_requests(vocab, dtype, chain):
    """No requests and a vocabulary of several parts: what lies behind the only entry of qo_indptr is not the call's, and it has
    no workspace.  Every row gets no token."""
    from deserve_amd.draft_ops import verify_drafts

    print("[case] rows without requests", vocab, dtype, chain, flush=True)
    target, draft, _, uniforms = make(6, [9], vocab, dtype)
    longer = dev([0, 5, 9])
    got = verify_drafts(target, dev(np.arange(9)), dev(uniforms, np.float32), longer[:1], draft_probs=draft if chain else None)
    assert got.counts.numel() == 0
    assert got.path.tolist() == [-1] * 9 and got.tokens.tolist() == [-1] * 9
    assert longer.tolist() == [0, 5, 9]
