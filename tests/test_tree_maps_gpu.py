"""Tree maps and commits (engine/hip_tree.py tree_maps, commit_tokens; sipa_tree_maps, sipa_commit_tokens) against plain
restatements: every value equal, and nothing outside touched."""

import numpy as np
import pytest
import torch

from engine.hip_tree import TreeMaps, commit_tokens, tree_maps
from tree_cases import ancestor_sets, mask_tensor, random_parents

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


class Maps:
    def __init__(self, seqs, block=16, seed=0, chain=False, capacity=0):
        rng = np.random.RandomState(seed)
        self.seqs, self.B = seqs, block
        S = len(seqs)
        self.width = max(max(-(-(c + n) // block) for c, n in seqs), 1)
        table = rng.randint(0, 100000, (S + 5, self.width + 3))
        self.rows = rng.permutation(S + 5)[:S]
        self.parents = [random_parents(n, rng, chain) for _, n in seqs]
        flat = [p for ps in self.parents for p in ps]
        self.T = len(flat)
        self.max_nodes = max(max(n for _, n in seqs), 1)
        self.table_cpu = table
        self.table, self.rows_t = i32(table), i32(self.rows)
        self.starts, self.counts = i32([c for c, _ in seqs]), i32([n for _, n in seqs])
        self.parents_t = i32(flat + [-1] * capacity)

    def run(self, **kw):
        return tree_maps(self.table, self.rows_t, self.starts, self.counts, self.parents_t, self.B, self.width,
                         self.max_nodes, **kw)

    def check(self, m: TreeMaps):
        pos, slots, at, qs = [], [], 0, [0]
        sets = []
        bt = np.full((len(self.seqs), self.width), -1)
        for i, (c, n) in enumerate(self.seqs):
            row = self.table_cpu[self.rows[i]]
            mine = ancestor_sets(self.parents[i])
            sets += mine
            pos += [c + len(a) - 1 for a in mine]
            slots += [int(row[p // self.B]) * self.B + p % self.B for p in range(c, c + n)]
            nb = -(-(c + n) // self.B)
            bt[i, :nb] = row[:nb]
            at += n
            qs.append(at)
        T = self.T
        assert m.query_starts.tolist() == qs
        assert m.positions[:T].tolist() == pos
        assert m.slots[:T].tolist() == slots
        assert m.slot_blocks[:T].tolist() == [s // self.B for s in slots]
        assert m.slot_offsets[:T].tolist() == [s % self.B for s in slots]
        assert m.last_rows.tolist() == [q - 1 for q in qs[1:]]
        assert m.context_lens.tolist() == [c + n for c, n in self.seqs]
        assert m.block_tables.tolist() == bt.tolist()
        assert torch.equal(m.masks[:T].cpu(), mask_tensor(sets, m.masks.shape[1]))


@pytest.mark.parametrize("block", [16, 32, 64, 7])
@pytest.mark.parametrize("seqs", [[(0, 1)], [(1000, 5)], [(15, 1), (16, 2), (17, 64), (0, 65), (3, 128)],
                                  [(5, 256), (9, 255), (100, 129), (0, 1)], [(7, 200), (8, 200), (9, 200)]],
                         ids=["one", "small", "words", "largest", "across"])
def test_maps_match(seqs, block):
    for seed, chain in ((0, False), (1, True)):
        m = Maps(seqs, block, seed, chain)
        m.check(m.run())


@pytest.mark.parametrize("S", [2, 255, 256, 257, 1000, 8192])
def test_many_sequences(S):
    rng = np.random.RandomState(S)
    m = Maps([(int(rng.randint(0, 90)), int(rng.randint(1, 5))) for _ in range(S)], seed=S)
    m.check(m.run())


def test_sequences_without_nodes():
    m = Maps([(5, 0), (3, 4), (9, 0), (0, 0), (2, 3), (7, 0)], seed=4)
    m.check(m.run())


def test_rows_behind_the_last_sequence_stay():
    m = Maps([(5, 3), (70, 9)], seed=5, capacity=300)
    T = m.T + 300
    out = TreeMaps(*(torch.full((T,), -5, dtype=torch.int64, device="cuda") for _ in range(4)),
                   torch.zeros(2, dtype=torch.int64, device="cuda"), i32([0] * 3), i32([0] * 2),
                   torch.zeros(2, m.width, dtype=torch.int32, device="cuda"),
                   torch.full((T, 1), -5, dtype=torch.int64, device="cuda"))
    got = m.run(out=out)
    assert got is out
    m.check(out)
    for t in out[:4]:
        assert (t[m.T:] == -5).all()
    assert (out.masks[m.T:] == -5).all()


def test_bad_parents_and_rows_stay_inside():
    """A parent that is not before its node ends the chain; table rows and columns are clamped."""
    m = Maps([(5, 4), (3, 3)], seed=6)
    m.parents_t.copy_(i32([3, 0, 2, -9, 5, 0, 7]))
    m.parents = [[-1, 0, -1, -1], [-1, 0, -1]]
    m.check(m.run())
    m.rows_t.fill_(1000)
    m.starts.fill_(1 << 30)
    m.run()  # entries of the table's last row and column
    torch.cuda.synchronize()


def test_maps_in_a_graph():
    m = Maps([(5, 3), (70, 9), (33, 1)], seed=7)
    out = m.run()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        m.run(out=out)
    for seed in (8, 9, 10):
        o = Maps([(seed, 4), (2 * seed, 2), (3 * seed, 7)], seed=seed)
        for a, b in ((m.starts, o.starts), (m.counts, o.counts), (m.parents_t, o.parents_t), (m.rows_t, o.rows_t)):
            a.copy_(b)
        m.table[:, :o.table.shape[1]].copy_(o.table[:, :m.table.shape[1]])
        g.replay()
        torch.cuda.synchronize()
        o.width, o.table_cpu = m.width, m.table.cpu().numpy()
        o.check(out)


def test_map_refusals():
    m = Maps([(5, 3), (70, 9)], seed=11)

    def refused(table=m.table, rows=m.rows_t, starts=m.starts, counts=m.counts, parents=m.parents_t, block=16,
                width=m.width, nodes=9, **kw):
        with pytest.raises(ValueError):
            tree_maps(table, rows, starts, counts, parents, block, width, nodes, **kw)

    refused(table=m.table.long())
    refused(table=m.table.t())
    refused(rows=m.rows_t[:1])
    refused(starts=m.starts.long())
    refused(parents=m.parents_t[::2])
    refused(parents=m.parents_t[:0])
    refused(nodes=0)
    refused(nodes=257)
    refused(width=0)
    refused(block=0)
    refused(parents=m.parents_t.cpu())
    out = m.run()
    refused(out=out._replace(masks=out.masks.int()))
    refused(out=out._replace(slots=out.slots[:-1]))
    big = torch.zeros(8193, dtype=torch.int32, device="cuda")
    refused(rows=big, starts=big, counts=big)


# ---- commits -------------------------------------------------------------------------------------------------------


class Commit:
    def __init__(self, starts, accepted, dtype=torch.bfloat16, layers=3, heads=2, D=64, block=16, seed=0):
        g = torch.Generator().manual_seed(seed)
        rng = np.random.RandomState(seed)
        self.starts, self.accepted, self.B = starts, accepted, block
        need = [-(-(s + max(a, default=0) + 1) // block) for s, a in zip(starts, accepted)]
        N = sum(need) + 2
        ids = rng.permutation(N)
        self.tables, at = [], 0
        for k in need:
            self.tables.append(ids[at:at + k])
            at += k
        bt = np.full((len(starts), max(need)), -1)
        for i, t in enumerate(self.tables):
            bt[i, :len(t)] = t
        shape = (layers, heads, N, block, D)
        self.ks = self.vs = None
        if dtype is torch.int8:
            self.k, self.v = (torch.randint(-127, 128, shape, generator=g, dtype=torch.int8).cuda() for _ in range(2))
            self.ks, self.vs = (torch.rand(shape[:4], generator=g).half().cuda() for _ in range(2))
        else:
            self.k, self.v = (torch.randn(shape, generator=g).to(dtype).cuda() for _ in range(2))
        A = max(max(len(a) for a in accepted), 1)
        self.bt, self.starts_t = i32(bt), i32(starts)
        self.acc = i32([list(a) + [-1] * (A - len(a)) for a in accepted])
        self.num = i32([len(a) for a in accepted])

    def expected(self):
        out = [t.cpu().clone() if t is not None else None for t in (self.k, self.v, self.ks, self.vs)]
        for s, a, table in zip(self.starts, self.accepted, self.tables):
            for i, node in enumerate(a):
                p, q = s + i, s + node
                for t in out:
                    if t is not None:
                        t[:, :, table[p // self.B], p % self.B] = t[:, :, table[q // self.B], q % self.B].clone()
        return out

    def run(self):
        commit_tokens(self.k, self.v, self.bt, self.starts_t, self.acc, self.num, k_scale=self.ks, v_scale=self.vs)

    def check(self, want):
        for t, w in zip((self.k, self.v, self.ks, self.vs), want):
            if w is not None:
                assert torch.equal(t.cpu(), w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int8, torch.float32])
@pytest.mark.parametrize("D,block", [(64, 16), (128, 16), (64, 32), (16, 7)])
def test_commit_moves_the_accepted_path(dtype, D, block):
    # chains whose sources are other moves' destinations, gaps, nothing to do, nothing accepted, more than one batch of moves
    paths = [[0, 2, 3, 4, 9], [1, 2, 3], [0, 1, 2], [], [0], list(range(1, 30)), [0, 5, 6, 7] + list(range(20, 40))]
    c = Commit([15, 0, 33, 7, 100, 3, 14], paths, dtype, D=D, block=block, seed=D)
    want = c.expected()
    c.run()
    c.check(want)


def test_commit_of_longest_path_and_layers_apart():
    c = Commit([9, 4], [list(range(3, 250)), [0, 255]], layers=2, seed=3)
    both = torch.stack([c.k, c.v], 1)  # K and V of a layer side by side: the layers of each lie apart
    c.k, c.v = both[:, 0], both[:, 1]
    want = c.expected()
    c.run()
    c.check(want)


def test_commit_clamps_indices():
    c = Commit([5], [[0, 2]], seed=4)
    c.bt.fill_(1 << 20)
    c.starts_t.fill_(1 << 28)
    c.num.fill_(100)
    c.run()
    torch.cuda.synchronize()


def test_commit_refusals():
    c = Commit([5, 9], [[0, 2], [1]], seed=5)
    i = Commit([5, 9], [[0, 2], [1]], torch.int8, seed=5)

    def refused(k=c.k, v=c.v, bt=c.bt, starts=c.starts_t, acc=c.acc, num=c.num, **kw):
        before = k.clone()
        with pytest.raises(ValueError):
            commit_tokens(k, v, bt, starts, acc, num, **kw)
        assert torch.equal(k, before)

    refused(v=c.v[:, :1])
    refused(k=c.k.transpose(3, 4), v=c.v.transpose(3, 4))
    refused(k=i.k, v=i.v)
    refused(k_scale=i.ks, v_scale=i.vs)
    refused(k=i.k, v=i.v, k_scale=i.ks, v_scale=i.vs[:, :1])
    refused(k=i.k, v=i.v, k_scale=i.ks.float(), v_scale=i.vs.float())
    refused(k=i.k[..., :8].contiguous(), v=i.v[..., :8].contiguous(), k_scale=i.ks, v_scale=i.vs)  # 8-byte rows
    refused(bt=c.bt[:1])
    refused(starts=c.starts_t.long())
    refused(acc=c.acc.long())
    refused(num=c.num[:1])
    refused(starts=c.starts_t.cpu())
