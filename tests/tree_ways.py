"""A round of a tiny model whose accepted way is known beforehand, and how far the logits of a wrong tree are from those of the right one."""
import random

import torch

from mllm_b200 import ops
from tree_cases import Round, ways_of

TREE, WAY = [-1, 0, 0, 1, 1, 3, 2, 2, 6], [2, 6, 8]


def round_of(preset, device, dtype, **kw):
    r = Round(preset, device, dtype, **kw)
    g = random.Random(11)
    ids = [g.randrange(r.mr.vocab_size) for _ in range(40)]
    row, logits = r.prompt(ids)
    seen = ids + [int(logits.float().argmax())]
    tokens = [seen[-1]] + [g.randrange(r.mr.vocab_size) for _ in TREE[1:]]
    for k, node in enumerate(WAY):          # this way is what the model itself would say
        tokens[node] = int(r.plain(seen + [tokens[i] for i in WAY[:k]]).float().argmax())
    return r, row, seen, tokens


def accepted_way(preset, device, dtype, **kw):
    """The walk of greedy verification is the planned way, node by node."""
    r, row, seen, tokens = round_of(preset, device, dtype, **kw)
    fb, logits = r.tree([row], [40], [tokens], [TREE])
    last = int(r.plain(seen + [tokens[i] for i in WAY]).float().argmax())
    f = lambda x, n: torch.full((n,), x, device=r.dev)  # noqa: E731
    path, out, counts = ops.tree_speculative_sample(
        logits, torch.tensor(tokens, device=r.dev), fb.tree_parents, fb.extend_seq_lens, fb.extend_start_loc, f(0.0, 1),
        torch.zeros(1, dtype=torch.int32, device=r.dev), f(1.0, 1), None, f(0.5, len(TREE)), f(0.5, 1), 6)
    assert path[0].tolist() == [0] + WAY + [-1, -1]
    assert out[0].tolist() == [tokens[i] for i in WAY] + [last, -1, -1]
    assert int(counts[0]) == 4
    ops.check_status()


def errors(preset, device, dtype, **kw):
    """Relative errors (2-norms) of the nodes' logits against the same tokens as plain prompts: of the tree, and of the nodes that a wrong
    parent moves, with one parent changed."""
    r, row, seen, tokens = round_of(preset, device, dtype, **kw)
    plain = [r.plain(seen[:-1] + [tokens[i] for i in way]).double() for way in ways_of(TREE)]

    def of(tree):
        _, logits = r.tree([row], [40], [tokens], [tree])
        return [((logits[i].double() - p).norm() / p.norm()).item() for i, p in enumerate(plain)]

    right = of(TREE)
    wrong = []
    for node, parent in ((3, 2), (6, 1), (4, 0), (5, 4)):        # a sibling instead, a level up, a cousin
        changed = list(TREE)
        changed[node] = parent
        wrong.append(of(changed)[node])
    ops.check_status()
    return right, wrong
