"""Taking over a verified draft tree on the GPU: path, counts, answers and every byte of the caches
against a plain walk on the CPU, and its refusals. All results are whole numbers or copies: equal, no tolerance."""

import random
from types import SimpleNamespace

import pytest
import torch

from babyvllm.kernels.tree_commit import commit_draft_tree
from tests._cases import cdiv, python_path

pytestmark = pytest.mark.gpu
PAGE = 16


def build(specs, layers=3, hkv=2, d=64, seed=0):
    """specs: (context, parents, draft tokens, answers) per sequence."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    seq = [c + len(p) for c, p, *_ in specs]
    pages = [cdiv(n, PAGE) for n in seq]
    total = sum(pages) + 2
    perm = torch.randperm(total, device="cuda", generator=g).tolist()
    width = max(max(pages), 1)
    tables = [[perm.pop() for _ in range(n)] + [-1] * (width - n) for n in pages]
    # Any bit pattern moves: NaNs and infinities among them.
    stack = torch.randint(-32768, 32768, (layers, 2, total, PAGE, hkv, d), device="cuda", dtype=torch.int16,
                          generator=g).view(torch.bfloat16)
    qsl = [0]
    for _, p, *_ in specs:
        qsl.append(qsl[-1] + len(p))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    i64 = lambda v: torch.tensor(v, dtype=torch.int64, device="cuda")  # noqa: E731
    md = SimpleNamespace(block_tables=i32(tables), query_start_loc=i32(qsl), context_lens=i32([c for c, *_ in specs]),
                         max_query_len=max(len(p) for _, p, *_ in specs))
    flat = lambda k: [x for s in specs for x in s[k]]  # noqa: E731
    return stack, md, i64(flat(2)), i64(flat(3)), i32(flat(1))


def walk(specs, stack, md, max_path):
    """(path, accepted, following, caches) by the definition."""
    bits = stack.cpu().view(torch.int16).clone()
    tables = md.block_tables.tolist()
    paths, counts, answers = [], [], []
    for s, (ctx, parents, draft, target) in enumerate(specs):
        path = [0] if parents else []
        while path and len(path) < max_path:
            nxt = [c for c in range(path[-1] + 1, len(parents))
                   if parents[c] == path[-1] and draft[c] == target[path[-1]]]
            if not nxt:
                break
            path.append(nxt[0])
        at = lambda i: (tables[s][(ctx + i) // PAGE], (ctx + i) % PAGE)  # noqa: E731
        rows = [bits[:, :, at(n)[0], at(n)[1]].clone() for n in path]
        for i, row in enumerate(rows):
            bits[:, :, at(i)[0], at(i)[1]] = row
        paths.append(path + [-1] * (max_path - len(path)))
        counts.append(len(path))
        answers.append(target[path[-1]] if path else -1)
    return torch.tensor(paths, dtype=torch.int32), torch.tensor(counts, dtype=torch.int32), torch.tensor(answers), bits


def check(specs, max_path=None, **kw):
    stack, md, draft, target, parents = build(specs, **kw)
    bound = max(1, md.max_query_len) if max_path is None else max_path
    path, counts, answers, bits = walk(specs, stack, md, bound)
    got = commit_draft_tree(list(stack.unbind(0)), md, draft, target, parents, max_path)
    assert torch.equal(got[0].cpu(), path) and torch.equal(got[1].cpu(), counts) and torch.equal(got[2].cpu(), answers)
    assert torch.equal(stack.cpu().view(torch.int16), bits)
    return path


def random_spec(rng, ctx, n, accept, branch=6, vocab=50):
    """A tree whose answers follow a drafted child with probability ``accept``; few tokens, so equal siblings occur."""
    parents = [-1] + [rng.randrange(max(0, i - branch), i) for i in range(1, n)]
    draft = [rng.randrange(vocab) for _ in range(n)]
    target = []
    for i in range(n):
        kids = [c for c in range(n) if parents[c] == i]
        target.append(draft[rng.choice(kids)] if kids and rng.random() < accept else vocab + rng.randrange(9))
    return ctx, parents, draft, target


@pytest.mark.parametrize("hkv,d,layers", [(2, 64, 1), (4, 128, 5), (1, 64, 3), (3, 128, 2)])
def test_random_trees(hkv, d, layers):
    rng = random.Random(hkv)
    specs = [random_spec(rng, rng.choice([0, 1, 15, 16, 17, 100]), rng.choice([1, 2, 9, 33, 64, 65, 140]),
                         rng.choice([0.0, 0.7, 1.0])) for _ in range(40)]
    check(specs, layers=layers, hkv=hkv, d=d)


def test_chains_accepted_whole_to_a_bound_and_not_at_all():
    n = 200
    chain = (37, list(range(-1, n - 1)), list(range(n)), list(range(1, n + 1)))
    assert (check([chain])[0] == torch.arange(n)).all()
    assert check([chain], max_path=1)[0].tolist() == [0]
    assert check([chain], max_path=7)[0].tolist() == list(range(7))
    assert check([(5, [-1, 0, 1], [1, 2, 3], [9, 9, 9])])[0].tolist() == [0, -1, -1]


def test_paths_whose_rows_overlap_their_destinations():
    # A long path shifted by one: every destination is the source of the next move.
    n = 130
    parents = [-1, 0, 0] + list(range(2, n - 1))
    draft = [7] * 2 + list(range(100, 100 + n - 2))
    target = [100, 0] + list(range(101, 101 + n - 2))
    path = check([(9, parents, draft, target)])[0].tolist()
    assert path[:4] == [0, 2, 3, 4] and path[n - 2] == n - 1


def test_equal_siblings_take_the_first_and_sequences_may_be_empty():
    tree = ([-1, 0, 0, 0, 2, 1], [0, 5, 5, 6, 8, 8], [5, 8, 8, 0, 1, 3])
    path = check([(10, *tree), (4, [], [], []), (30, *tree)])
    assert path[0].tolist() == [0, 1, 5, -1, -1, -1] and (path[1] == -1).all()


def test_many_layers_and_no_layers():
    rng = random.Random(1)
    specs = [random_spec(rng, 20, 30, 0.9) for _ in range(3)]
    check(specs, layers=70, hkv=1)  # more than one launch holds
    stack, md, draft, target, parents = build(specs)
    path, counts, answers, _ = walk(specs, stack, md, md.max_query_len)
    got = commit_draft_tree([], md, draft, target, parents)
    assert torch.equal(got[0].cpu(), path) and torch.equal(got[1].cpu(), counts) and torch.equal(got[2].cpu(), answers)


def test_head_major_caches_and_the_python_path(monkeypatch):
    rng = random.Random(2)
    specs = [random_spec(rng, rng.randrange(50), 40, 0.9) for _ in range(5)]
    stack, md, draft, target, parents = build(specs)
    *_, bits = walk(specs, stack, md, md.max_query_len)
    caches = [c.permute(0, 1, 3, 2, 4).contiguous().permute(0, 1, 3, 2, 4) for c in stack.unbind(0)]
    commit_draft_tree(caches, md, draft, target, parents)
    assert torch.equal(torch.stack(caches).cpu().view(torch.int16), bits)
    python_path(monkeypatch)
    check(specs)
    check(specs, max_path=3)


def test_tables_that_lead_out_of_the_pool_move_nothing_there():
    n = 20
    chain = (14, [-1, 0, 0] + list(range(2, n - 1)), [9, 9] + list(range(n - 2)), [0, 0] + list(range(1, n - 1)))
    stack, md, draft, target, parents = build([chain])
    md.block_tables[0, 1] = 1 << 20
    before = stack.clone()
    path, counts, _ = commit_draft_tree(list(stack.unbind(0)), md, draft, target, parents)
    assert counts.item() == n - 1
    # Node 2 lies on the page that is not there: nothing of the first page changes.
    page = int(md.block_tables[0, 0])
    assert torch.equal(stack[:, :, page].view(torch.int16), before[:, :, page].view(torch.int16))


def test_in_a_graph_that_is_replayed_with_other_answers():
    rng = random.Random(3)
    sets = [[random_spec(rng, 33, 25, 0.95) for _ in range(4)] for _ in range(3)]
    stack, md, draft, target, parents = build(sets[0])
    caches = list(stack.unbind(0))
    commit_draft_tree(caches, md, draft, target, parents)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = commit_draft_tree(caches, md, draft, target, parents)
    for i in (1, 0, 2, 1):
        fresh, _, d, t, p = build(sets[i], seed=i)
        stack.copy_(fresh)
        draft.copy_(d), target.copy_(t), parents.copy_(p)
        path, counts, answers, bits = walk(sets[i], stack, md, md.max_query_len)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0].cpu(), path) and torch.equal(got[1].cpu(), counts) and torch.equal(got[2].cpu(), answers)
        assert torch.equal(stack.cpu().view(torch.int16), bits)


def test_refusals():
    stack, md, draft, target, parents = build([(3, [-1, 0], [1, 2], [2, 3])])
    caches = list(stack.unbind(0))

    def refused(error, caches=caches, draft=draft, target=target, parents=parents, max_path=None, **changes):
        with pytest.raises(error):
            commit_draft_tree(caches, SimpleNamespace(**{**vars(md), **changes}), draft, target, parents, max_path)

    refused(TypeError, draft=draft.int())
    refused(TypeError, parents=parents.long())
    refused(ValueError, target=target[:1])
    refused(ValueError, parents=parents[:1])
    refused(ValueError, max_path=0)
    refused(ValueError, max_path=4097)
    refused(ValueError, query_start_loc=md.query_start_loc[:1])
    refused(ValueError, block_tables=md.block_tables[:0])
    refused(ValueError, caches=[caches[0], caches[1][:, :1]])
    refused(ValueError, caches=[caches[0][0]])
    refused(ValueError, caches=caches + caches[:1])  # moved twice at once
    refused(TypeError, caches=[caches[0].float()])
    refused(RuntimeError, caches=[caches[0].cpu()])
    refused(RuntimeError, draft=draft.cpu())
    refused(RuntimeError, caches=[c[:, :, :8].contiguous() for c in caches])
