"""The calls between the linears together: a decode with drafted tokens (p8x.tree_decode) gives what decoding token by token
does, and keeps its cache within the budget."""
import numpy as np
import pytest

import p8x
from p8x import tree_decode as td

pytestmark = pytest.mark.gpu
SMALL = dict(layers=2, hidden=512, heads=4, kv=2, head_dim=128, ffn=768, vocab=256, seed=3)


def close(a, b):
    # the sums of the attention and the norms are in another order, 2^-20 or so, which may move an activation to the next of
    # the linears' 127 steps a block; through two layers the logits may differ by some of such steps
    assert np.abs(a - b).max() <= 0.03 * np.abs(b).max(), np.abs(a - b).max() / np.abs(b).max()


def test_tree_equals_each_of_its_paths():
    m = td.Model(**SMALL)
    prompt = np.random.default_rng(0).integers(0, 256, 21).tolist()
    tokens, parents = [5, 9, 200, 9, 77, 1, 3], [-1, 0, 0, 1, 2, 4, 0]
    d = td.Decoder(m, 128)
    d.prompt(prompt)
    tree = d.forward(tokens, parents)
    for leaf in (3, 5, 6):
        path = [leaf]
        while parents[path[0]] >= 0:
            path.insert(0, parents[path[0]])
        one = td.Decoder(m, 128)
        one.prompt(prompt)
        for i in path:
            close(tree[i], one.forward([tokens[i]], [-1])[0])
            one.keep([0])
    d.keep([0, 2, 4])
    for L in d.layers:
        assert L["len"].to_numpy(np.int32, (1,))[0] == 24
        pos = L["pos"].to_numpy(np.int32, (2, d.max_len))[:, :24]
        assert (pos == np.arange(24)).all()
    after = d.forward([8], [-1])[0]
    one = td.Decoder(m, 128)
    one.prompt(prompt)
    for t in (5, 200, 77):
        one.forward([t], [-1])
        one.keep([0])
    close(after, one.forward([8], [-1])[0])


def test_budget():
    """every head keeps the first and last positions and one slot a position, its scores the sum that it was given"""
    m = td.Model(**SMALL)
    d = td.Decoder(m, 48, n_sink=3, n_recent=10, page=16, decay=1.0)
    rng = np.random.default_rng(1)
    seen = 0
    for n in (8, 8, 8, 8, 8, 8, 3, 5, 8, 1, 2):
        d.forward(rng.integers(0, 256, n).tolist(), range(-1, n - 1))
        d.keep(range(n))
        seen += n
        for L in d.layers:
            used = min(48, seen)
            assert L["len"].to_numpy(np.int32, (1,))[0] == used == d.length
            pos, score = (L[k].to_numpy(t, (2, d.max_len))[:, :used] for k, t in (("pos", np.int32), ("score", np.float32)))
            for h in range(2):
                assert len(set(pos[h])) == used
                assert set(range(3)) | set(range(max(0, seen - 10), seen)) <= set(pos[h].tolist())
            if seen <= 48:   # nothing cut yet: every token gave each of its heads a weight of one
                assert np.allclose(score.sum(axis=1), seen * m.heads / m.kv, rtol=1e-4)


def test_drafts_do_not_change_the_tokens():
    """guesses taken from the greedy sequence itself, some of them spoiled"""
    m = td.Model(**SMALL)
    prompt = [7, 8, 9, 10]
    want, steps = td.generate(td.Decoder(m, 256), prompt, 40, drafts=1)
    assert steps == 39

    def propose(known, limit):
        at = len(known) - len(prompt)
        follow = want[at:at + 4]
        if at % 3 == 0 and len(follow) > 2:
            follow[2] = (follow[2] + 1) % m.vocab
        # the true path and a wrong sibling of its first token
        tokens, parents = [known[-1]] + follow + [(follow[0] + 5) % m.vocab] if follow else [known[-1]], [-1]
        parents += list(range(len(follow))) + ([0] if follow else [])
        return tokens, parents
    got, steps = td.generate(td.Decoder(m, 256), prompt, 40, propose=propose)
    assert got == want and steps < 20
