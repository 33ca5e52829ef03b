"""GPU tests of the drafted-tree metadata on caches whose rows are not the tokens that
their sequences have seen (marked ``gpu``): the operator against its 64-bit
restatement, and a drafting loop on caches that are cut, against attention over plain
lists of tokens at absolute positions.

Tolerance of the loop: an angle of up to 150 is off by 150 * 2^-24 in float32, for the
query and for the key, so a score by 2 * 150 * 2^-24 * sum |q_e k_e| * scale, with both
members of a rotated pair less than 2 * 25 (normal queries of deviation 2 and keys of
1): 9e-4.  Its float32 sum adds (E + 8) * 2^-24 * 25 = 2e-4.  A weight is off by a
factor exp(2 * 1.1e-3), an output by that times |v| < 5: 1.2e-2.
"""
import pytest
import torch

from oracle import tree_cache_oracle as TO
from test_gpu_tree_cache import E, SCALE, dv, meta_inputs  # noqa: F401

pytestmark = pytest.mark.gpu

TOL = 1.2e-2


def check_counts(dv, gpu, fl, order, parents, inv, **counts):
    want = TO.metadata(fl, order, parents, inv, 1.0, **counts)
    got = [t.cpu() for t in dv.dvattn_tree_metadata(fl.to(gpu), order.to(gpu), parents.to(gpu), inv.to(gpu),
                                                    **{k: v.to(gpu) for k, v in counts.items()})]
    for i in (0, 3, 4):
        assert torch.equal(got[i], want[i])
    for i in (1, 2):  # cosf and sinf: a few units in the last place of values up to 1
        assert (got[i].double() - want[i]).abs().max().item() <= 4 * 2.0 ** -24
    return got


@pytest.mark.parametrize("W,F,S,R", [(1, 1, 1, 128), (3, 2, 9, 64), (2, 5, 70, 20)])
def test_dropped_tokens_count_for_positions_only(dv, gpu, W, F, S, R):  # noqa: F811
    fl, order, parents, inv = meta_inputs(W, F, S, R, seed=S)
    g = torch.Generator().manual_seed(F)
    dropped = torch.randint(0, 3000, (W, F), generator=g).to(torch.int32)
    got = check_counts(dv, gpu, fl, order, parents, inv, dropped=dropped)
    plain = [t.cpu() for t in dv.dvattn_tree_metadata(*(t.to(gpu) for t in (fl, order, parents, inv)))]
    assert all(torch.equal(got[i], plain[i]) for i in (0, 3, 4)) and not torch.equal(got[2], plain[2])
    check_counts(dv, gpu, fl, order, parents, inv, dropped=torch.zeros_like(dropped))


@pytest.mark.parametrize("W,F,S,R", [(1, 1, 1, 128), (4, 1, 9, 64), (3, 5, 70, 20)])
def test_committed_rows_of_each_sequence(dv, gpu, W, F, S, R):  # noqa: F811
    """Rows below zero count as none; rows of sequences all alike are the lengths' own."""
    fl, order, parents, inv = meta_inputs(W, F, S, R, seed=S + 1)
    g = torch.Generator().manual_seed(F)
    committed = torch.randint(-3, 400, (W, F), generator=g).to(torch.int32)
    dropped = torch.randint(0, 50, (W, F), generator=g).to(torch.int32)
    check_counts(dv, gpu, fl, order, parents, inv, committed=committed)
    check_counts(dv, gpu, fl, order, parents, inv, committed=committed, dropped=dropped)
    own = torch.zeros(F, dtype=torch.int32)
    own[order[:, -1].long()] = S
    alike = (fl - own).clamp(min=0).expand(W, F).contiguous()
    got = check_counts(dv, gpu, fl, order, parents, inv, committed=alike)
    plain = dv.dvattn_tree_metadata(*(t.to(gpu) for t in (fl, order, parents, inv)))
    assert all(torch.equal(a, b.cpu()) for a, b in zip(got, plain))


def test_counts_refused(dv, gpu):  # noqa: F811
    args = [t.to(gpu) for t in meta_inputs(2, 3, 4, 64, seed=1)]
    good = torch.zeros(2, 3, dtype=torch.int32, device=gpu)
    for name in ("dropped", "committed"):
        for bad, text in ((good[:1], "must be"), (good.long(), "int32"), (good.t().contiguous().t(), "contiguous")):
            with pytest.raises(RuntimeError, match=text):
                dv.dvattn_tree_metadata(*args, **{name: bad})
        with pytest.raises(RuntimeError):
            dv.dvattn_tree_metadata(*args, **{name: good.cpu()})


class Loop:
    """Sequences of a prompt (view 0) and tokens of their own (view 1), whose own rows
    each KV head may have cut; `tokens[w][h]` lists what the cache should hold:
    (absolute position, key before its rotation, value)."""

    def __init__(self, dv, gpu, prompt, seed):
        self.dv, self.gpu, self.prompt = dv, gpu, prompt
        self.g = torch.Generator().manual_seed(seed)
        self.W, self.Hkv, self.R, self.bs = 2, 2, 64, 16
        self.inv = (1e4 ** (-torch.arange(0, self.R, 2, dtype=torch.float64) / self.R)).float()
        maxB = 12
        P = self.W * maxB
        self.bt = torch.randperm(P, generator=self.g).to(torch.int32).reshape(self.W, maxB).to(gpu)
        self.kc, self.vc = (torch.zeros(P, self.bs, self.Hkv, E, device=gpu) for _ in range(2))
        self.tokens = [[[] for _ in range(self.Hkv)] for _ in range(self.W)]
        self.order = torch.tensor([[0, 1]] * self.W, dtype=torch.int32, device=gpu)
        self.dropped = torch.zeros(self.W, 2, dtype=torch.int32, device=gpu)

    def rope(self, x, pos):
        a = float(pos) * self.inv.double()
        h = self.R // 2
        y = x.clone()
        y[..., :h] = x[..., :h] * torch.cos(a) - x[..., h:2 * h] * torch.sin(a)
        y[..., h:2 * h] = x[..., h:2 * h] * torch.cos(a) + x[..., :h] * torch.sin(a)
        return y

    def append(self, rows, cos, sin, at):
        """New tokens in stream rows [W,S] with rotary tables [W,S,R]; at [W][S]: absolute positions."""
        S = rows.shape[1]
        k, v = (torch.randn(self.W, self.Hkv, S, E, generator=self.g) for _ in range(2))
        self.dv.dvattn_paged_kv_append(k.to(self.gpu), v.to(self.gpu), rows, cos, sin, self.kc, self.vc, self.bt)
        return [[[(at[w][s], k[w, h, s].double(), v[w, h, s].double()) for s in range(S)] for h in range(self.Hkv)]
                for w in range(self.W)]

    def fill(self, first, n, absolute):
        """n tokens of a view that starts at row `first` and position `absolute`."""
        ang = torch.arange(n, dtype=torch.float32)[:, None] * self.inv
        ang = torch.cat([ang, ang], -1).expand(self.W, n, self.R).to(self.gpu)
        rows = (first + torch.arange(n, dtype=torch.int32)).repeat(self.W, 1).to(self.gpu)
        new = self.append(rows, torch.cos(ang), torch.sin(ang), [list(range(absolute, absolute + n))] * self.W)
        for w in range(self.W):
            for h in range(self.Hkv):
                self.tokens[w][h] += new[w][h]

    def cut(self, held, budget):
        """Own rows down to the budget, by random weights; held [W]."""
        mass = torch.rand(self.W, self.Hkv, self.bt.shape[1] * self.bs, generator=self.g).to(self.gpu)
        first = torch.full((self.W,), self.prompt, dtype=torch.int32, device=self.gpu)
        lengths = held.to(torch.int32).to(self.gpu)
        rows = self.dv.dvattn_kv_select(mass, first, lengths, budget, 2, 5)
        self.dv.dvattn_paged_kv_compact(rows, first, self.kc, self.vc, self.bt, mass=mass, lengths=lengths)
        self.dropped[:, 1] += lengths - torch.clamp(lengths, max=budget)
        for w in range(self.W):
            for h in range(self.Hkv):
                own = self.tokens[w][h][self.prompt:]
                self.tokens[w][h][self.prompt:] = [own[i] for i in rows[w, h].tolist() if i >= 0]
        return torch.clamp(held, max=budget)

    def draft(self, parents, fl, next_position, **counts):
        """One drafted step; next_position [W]: where a child of the committed tokens stands."""
        W, S = parents.shape
        dv, gpu = self.dv, self.gpu  # noqa: F811
        fl = torch.tensor(fl, dtype=torch.int32, device=gpu)
        loc, cos, sin, views, first = dv.dvattn_tree_metadata(fl, self.order, parents.to(gpu), self.inv.to(gpu),
                                                              dropped=self.dropped, **counts)
        depth = [[len(TO.path(parents[w], s) or [0]) - 1 for s in range(S)] for w in range(W)]
        at = [[next_position[w] + d for d in depth[w]] for w in range(W)]
        rows = first[:, None] + torch.arange(S, dtype=torch.int32, device=gpu)
        w_of = torch.arange(W, device=gpu)
        new = self.append(rows, cos[views.long(), w_of], sin[views.long(), w_of], at)
        q = torch.randn(W, 16 * self.Hkv, S, E, generator=self.g) * 2
        out = dv.dvattn_tree_paged_sdpa(q.to(gpu), loc, cos, sin, fl, self.kc, self.vc, self.bt, parents.to(gpu), views,
                                        first, SCALE).cpu().double()
        weights = {}
        for w in range(W):
            for s in range(S):
                nodes = TO.path(parents[w], s)
                for h in range(self.Hkv):
                    got = out[w, 16 * h:16 * h + 16, s]
                    if nodes is None:
                        assert not got.any()
                        continue
                    seen = self.tokens[w][h] + [new[w][h][j] for j in sorted(nodes)]
                    k = torch.stack([self.rope(x[1], x[0]) for x in seen])
                    rq = self.rope(q[w, 16 * h:16 * h + 16, s].double(), at[w][s])
                    p = torch.softmax(rq @ k.T * SCALE, -1)
                    assert (got - p @ torch.stack([x[2] for x in seen])).abs().max() <= TOL, (w, s, h)
                    weights[w, h, s] = p.sum(0)
        return new, first, q, (loc, cos, sin, views, fl), weights

    def keep(self, accepted, new, first):
        """Accepted paths (ascending node indices) stay; returns their lengths [W]."""
        N = max(1, max(len(a) for a in accepted))
        path = torch.tensor([a + [-1] * (N - len(a)) for a in accepted], dtype=torch.int32, device=self.gpu)
        self.dv.dvattn_paged_kv_compact(path[:, None].contiguous(), first, self.kc, self.vc, self.bt)
        for w in range(self.W):
            for h in range(self.Hkv):
                self.tokens[w][h] += [new[w][h][j] for j in accepted[w]]
        return torch.tensor([len(a) for a in accepted])


PARENTS = torch.tensor([[-1, -1, 0, 0, 1, 3, -2], [-1, 0, 1, 1, 0, 3, 5]], dtype=torch.int32)


def test_drafting_on_caches_that_were_cut(dv, gpu):  # noqa: F811
    """Cut, draft, keep a path, draft, cut again, draft: the operator's own tables rotate
    the queries and the drafted keys."""
    loop = Loop(dv, gpu, prompt=37, seed=5)
    loop.fill(0, 37, 0)
    loop.fill(37, 60, 37)
    S = PARENTS.shape[1]
    held, position = torch.tensor([60, 60]), 97
    for budget in (30, None, 25):
        if budget:
            held = loop.cut(held, budget)
        n = int(held[0])
        new, first, *_ = loop.draft(PARENTS, [37, n + S], [position] * 2)
        assert first.tolist() == [37 + n] * 2
        held = held + loop.keep([[0, 3, 5], [0, 1, 3]], new, first)
        position += 3


def test_drafting_on_sequences_of_uneven_lengths(dv, gpu):  # noqa: F811
    """Accepted paths of different lengths, an own view that starts empty, and a cut that
    only the longer sequences need: each sequence's own rows, not the shared length."""
    loop = Loop(dv, gpu, prompt=20, seed=9)
    loop.fill(0, 20, 0)
    S = PARENTS.shape[1]
    held, position = torch.tensor([0, 0]), [20, 20]
    for accepted in ([[0, 3, 5], [0]], [[1, 4], [0, 1, 3, 5]], [[0], [0, 4]], [[], [0, 1, 2]], [[0, 2], [0, 1]]):
        if int(held.max()) > 8:
            held = loop.cut(held, 8)
        committed = torch.tensor([[20, int(n)] for n in held], dtype=torch.int32, device=gpu)
        new, first, *_ = loop.draft(PARENTS, [20, int(held.max()) + S], position, committed=committed)
        assert first.tolist() == [20 + int(n) for n in held]
        held = held + loop.keep(accepted, new, first)
        position = [p + len(a) for p, a in zip(position, accepted)]


def test_key_mass_of_accepted_tokens(dv, gpu):  # noqa: F811
    """The accepted tokens of a tree, passed as a causal chain once they are kept: every
    key collects the weights that the tree attention gave it.  A weight is off by a factor
    exp(2 * 1.1e-3), as above."""
    loop = Loop(dv, gpu, prompt=20, seed=3)
    loop.fill(0, 20, 0)
    loop.fill(20, 40, 20)
    W, S = PARENTS.shape
    held = loop.cut(torch.tensor([40, 40]), 25)
    committed = torch.tensor([[20, 25]] * W, dtype=torch.int32, device=gpu)
    for accepted in ([[0, 3, 5], [0]], [[1], [0, 1, 2]]):
        position = [20 + int(c) + int(d) for c, d in zip(committed[:, 1], loop.dropped[:, 1])]
        before = [len(loop.tokens[w][0]) for w in range(W)]
        new, first, q, (loc, cos, sin, views, fl), weights = loop.draft(
            PARENTS, [20, int(committed[:, 1].max()) + S], position, committed=committed)
        committed[:, 1] += loop.keep(accepted, new, first).to(torch.int32).to(gpu)
        F, N, R, Hq = 2, max(map(len, accepted)), cos.shape[3], q.shape[1]
        path = torch.tensor([a + [-1] * (N - len(a)) for a in accepted], dtype=torch.int32, device=gpu)[:, None]
        taken, take = path[:, 0] >= 0, path[:, 0].clamp(min=0).long()
        of = lambda t: t.gather(2, take.view(1, W, N, 1).expand(F, W, N, t.size(3)))  # noqa: E731
        seen = loc.gather(2, take.expand(F, W, N))
        seen[views.long(), torch.arange(W, device=gpu)] += 1 + torch.arange(N, dtype=torch.int32, device=gpu)
        seen = torch.where(taken, seen, -1)
        voters = q.to(gpu).gather(2, take.view(W, 1, N, 1).expand(W, Hq, N, E))
        mass = torch.rand(W, loop.Hkv, 80, generator=loop.g)
        got = dv.dvattn_paged_key_mass(mass.to(gpu), voters, seen, of(cos), of(sin), fl, loop.kc, loop.bt, SCALE,
                                       decay=0.5).cpu()
        want = mass.double() * 0.5
        for w in range(W):
            for h in range(loop.Hkv):
                for s in accepted[w]:
                    p = weights[w, h, s]
                    assert len(p) <= before[w] + len(accepted[w])
                    want[w, h, :len(p)] += p
        assert ((got - want).abs() <= 2.3e-3 * want).all()


def test_compaction_of_caches_that_share_rows(dv, gpu):  # noqa: F811
    """Refused where both certainly hold the same rows; keys and values side by side in one
    tensor are two caches."""
    rows = torch.tensor([[[1, 3]]], dtype=torch.int32, device=gpu)
    first, bt = torch.zeros(1, dtype=torch.int32, device=gpu), torch.tensor([[1, 0]], dtype=torch.int32, device=gpu)
    kv = torch.randn(2, 4, 2, 2, 64, generator=torch.Generator().manual_seed(1)).to(gpu)
    before = kv.clone()
    flat = kv.view(-1)
    one, behind = flat[:1024].view(2, 4, 1, 128), flat[512:1536].view(2, 4, 1, 128)
    for k, v in ((one, one), (one, behind), (kv[:, :, 0], kv[:, :, 0]), (kv[:, :, 0], kv[:, :, 0, :, :32])):
        with pytest.raises(RuntimeError, match="overlap"):
            dv.dvattn_paged_kv_compact(rows, first, k, v, bt)
    assert torch.equal(kv, before)
    dv.dvattn_paged_kv_compact(rows, first, kv[:, :, 0], kv[:, :, 1], bt)
    want = before.clone()
    want[1, 0], want[1, 1] = before[1, 1], before[1, 3]
    assert torch.equal(kv, want)
