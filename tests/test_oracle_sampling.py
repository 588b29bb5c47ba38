"""The sampling oracle on the CPU: the emitted tokens follow the target's distribution whatever the draft, the greedy limit
is the greedy walk, and known coins give known walks."""

import numpy as np
import pytest
import torch

from oracle import accept as oacc
from oracle import sampling as osm


def _frequencies(parents, draft, probs_of, runs=20000, seed=0):
    """First-token frequencies over ``runs`` walks of one tree; ``draft(rng, q)`` gives the drafted tokens of a run."""
    rng = np.random.default_rng(seed)
    vocab = 5
    logits = rng.normal(size=(len(parents), vocab)) * 1.5
    q = probs_of(rng, len(parents), vocab)
    first = np.zeros(vocab)
    for _ in range(runs):
        tokens, _ = osm.walk(logits, draft(rng, q), parents, rng.random(len(parents)), rng.random(), 0.8, q)
        first[tokens[0]] += 1
    return first / runs, osm.distribution(logits[0], 0.8)[0]


@pytest.mark.parametrize("parents", [[-1, 0, 1], [-1, 0, 0, 0]])
def test_drawn_children_leave_the_targets_distribution(parents):
    def probs(rng, rows, vocab):
        x = np.exp(rng.normal(size=(rows, vocab)) * 1.5)
        return x / x.sum(1, keepdims=True)

    def draft(rng, q):
        return np.array([0] + [rng.choice(q.shape[1], p=q[parents[r]]) for r in range(1, len(parents))])

    got, want = _frequencies(parents, draft, probs)
    assert np.abs(got - want).max() < 5 * np.sqrt(0.25 / 20000)  # five standard deviations of a frequency


def test_chosen_children_leave_the_targets_distribution():
    parents = [-1, 0, 0, 0]
    got, want = _frequencies(parents, lambda rng, q: np.array([0, 3, 1, 3]), lambda *a: None)  # one token twice
    assert np.abs(got - want).max() < 5 * np.sqrt(0.25 / 20000)


def test_temperature_zero_is_the_greedy_walk():
    gen = torch.Generator().manual_seed(4)
    parents = torch.tensor([[-1, 0, 0, 1, 1, 2, 3, 5]], dtype=torch.int32)
    for seed in range(50):
        logits = torch.randn(8, 6, generator=gen)
        drafted = torch.randint(0, 6, (8,), generator=gen)
        path, plen = torch.zeros(1, 8, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
        cu, idx = torch.tensor([0, 8]), torch.tensor([0])
        got, num = osm.sample_tree(logits, drafted, cu, idx, parents, torch.rand(8, generator=gen), torch.rand(1, generator=gen),
                                   torch.zeros(1), path, plen, 8)
        path2, plen2 = torch.zeros(1, 8, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
        want, num2 = oacc.accept_tree(logits.argmax(-1), drafted, cu.to(torch.int32), idx.to(torch.int32), parents, path2, plen2, 8)
        assert int(num[0]) == int(num2[0]) and got[0, : num[0]].tolist() == want[0, : int(num[0])].tolist()
        assert path[0, : num[0]].tolist() == path2[0, : num[0]].tolist()


def test_known_coins():
    logits = np.log(np.array([[0.5, 0.25, 0.125, 0.125]] * 3))
    parents, drafted = [-1, 0, 0], np.array([0, 1, 0])
    # row 1 (token 1): accepted iff coin < 1/4; then row 2 (token 0) against 1/2 of the 3/4 left
    assert osm.walk(logits, drafted, parents, [0, 0.2499, 0], 0.0, 1.0) == ([1, 0], [0, 1])
    assert osm.walk(logits, drafted, parents, [0, 0.2501, 0.666], 0.6, 1.0) == ([0, 1], [0, 2])
    # both rejected: tokens 2 and 3 are left, an eighth each
    assert osm.walk(logits, drafted, parents, [0, 0.2501, 0.667], 0.4999, 1.0) == ([2], [0])
    assert osm.walk(logits, drafted, parents, [0, 0.2501, 0.667], 0.5001, 1.0) == ([3], [0])


def test_rows_without_a_finite_maximum():
    bad = np.array([[-np.inf, -np.inf], [np.nan, 0.0], [np.inf, 0.0]])
    for row, want in zip(bad, (0, 0, 0)):
        p, single = osm.distribution(row, 1.0)
        assert single and int(p.argmax()) == want
