"""A round that drafts by sampling over quantized pages, its operators in the order in which they are used: page tables for the
rows to come, the prompts' rows into fp8 pages, then for every draft step slots, rotated rows, their page write, attention over the
pages and drawn tokens; the target's rows cut by the same rules, the sampled walk, and the pages that no accepted row needs given
back. Checked step by step against the oracles, and as one captured graph against the eager run."""

import numpy as np
import pytest
import torch

from conftest import announce
from oracle import page_tables as ora_tables
from oracle import rotary as ora_rotary
from oracle import row_attention as ora_rows
from oracle import sampling as ora_sampling

pytestmark = pytest.mark.gpu

REQS, ROWS, STEPS, HQ, HKV, DIM, PAGE, VOCAB, MOST = 3, 2, 2, 8, 2, 64, 16, 700, 8
WIDTH = 1 + ROWS * STEPS  # the root and the drafted nodes
PARENTS = [-1, 0, 0, 1, 2]  # two children of the root, then one of each


class Round:
    def __init__(self, dev, seed):
        gen = torch.Generator().manual_seed(seed)
        on = lambda t: t.to(dev)  # noqa: E731
        i32 = dict(dtype=torch.int32, device=dev)
        self.dev = dev
        self.lens = torch.randint(3, 60, (REQS,), generator=gen).int()
        self.context = on(self.lens)
        self.idx = torch.tensor([4, 0, 2], **i32)
        self.table, self.pages = torch.zeros(5, MOST, **i32), torch.zeros(5, **i32)
        self.free = on(torch.randperm(40, generator=gen).int())
        self.num_free = torch.tensor([40], **i32)
        shape = (40, PAGE, HKV, DIM)
        self.keys, self.values = (torch.zeros(shape, dtype=torch.float8_e4m3fn, device=dev) for _ in range(2))
        self.ks, self.vs = torch.zeros(40, HKV, device=dev), torch.zeros(40, HKV, device=dev)
        rows = lambda n, h: on(torch.randn(n, h, DIM, generator=gen).to(torch.bfloat16))  # noqa: E731
        self.longest = 60
        self.prompt = rows(REQS * self.longest, HKV), rows(REQS * self.longest, HKV)  # some rows of each are its prompt
        self.starts = on(torch.cat([torch.zeros(1), torch.cumsum(self.lens, 0)]).int())
        self.q, self.k, self.v = ([rows(REQS * ROWS, h) for _ in range(STEPS)] for h in (HQ, HKV, HKV))
        self.mix = on(torch.randint(0, HQ * DIM, (VOCAB,), generator=gen))
        self.noise = on(torch.randn(REQS * ROWS * STEPS, VOCAB, generator=gen))
        self.target = on(3 * torch.randn(REQS * WIDTH, VOCAB, generator=gen))
        self.coins = on(torch.rand(STEPS, REQS * ROWS, generator=gen))
        self.walk_coins, self.final = on(torch.rand(REQS * WIDTH, generator=gen)), on(torch.rand(REQS, generator=gen))
        self.t, self.top_k = on(torch.tensor([0.7, 1.0, 1.3])), torch.tensor([20, 0, 50], **i32)
        self.top_p = on(torch.tensor([0.9, 0.8, 1.0]))
        self.of_rows = torch.arange(REQS, **i32).repeat_interleave(ROWS)
        self.of_nodes = torch.arange(REQS, **i32).repeat_interleave(WIDTH)
        self.row_starts = torch.arange(0, REQS * ROWS + 1, ROWS, **i32)
        self.node_starts = torch.arange(0, REQS * WIDTH + 1, WIDTH, **i32)
        self.drafted = torch.zeros(REQS * WIDTH, dtype=torch.int64, device=dev)
        self.probs = torch.zeros(REQS * WIDTH, VOCAB, device=dev)
        self.parents = torch.tensor(PARENTS, device=dev)
        self.batch_table = torch.zeros(REQS, MOST, **i32)
        self.slots = [torch.zeros(REQS * ROWS, dtype=torch.int64, device=dev) for _ in range(STEPS)]

    def run(self):
        """One round; what it leaves, by name."""
        from eagle_harness.kernels.row_attention import RowsLaunch, rows_attention
        from eagle_harness.vllm.kv_pages import write_kv_pages
        from eagle_harness.vllm.page_tables import resize_tables, slot_maps
        from eagle_harness.vllm.rotary import rotate_rows
        from eagle_harness.vllm.sampling import draw_tokens, truncate_logits
        from eagle_harness.vllm.tree_accept import sample_tree

        dev, got = self.dev, {}
        resize_tables(self.table, self.pages, self.idx, self.context + ROWS * STEPS, self.free, self.num_free, PAGE)
        got["grown"] = self.table.clone(), self.pages.clone()
        slot_maps(self.table, self.pages, self.idx, self.context, self.row_starts, PAGE, slots=self.slots[0], batch_table=self.batch_table)
        prompts = torch.zeros(REQS, dtype=torch.int32, device=dev)
        write_kv_pages(*self.prompt, self.keys, self.values, self.ks, self.vs, self.batch_table, prompts, self.starts,
                       max_query_len=self.longest)
        got["steps"] = []
        ancestors = torch.zeros(REQS, ROWS, STEPS, dtype=torch.int32, device=dev)
        for step in range(STEPS):
            before = self.context + step * ROWS  # the nodes drafted so far lie behind the context
            slot_maps(self.table, self.pages, self.idx, before, self.row_starts, PAGE, slots=self.slots[step])
            positions = (self.context + step)[:, None].expand(-1, ROWS).reshape(-1)  # a node's position is its depth's
            q, k = rotate_rows(self.q[step], self.k[step], positions, self.frequencies, q_out=torch.empty_like(self.q[step]),
                               k_out=torch.empty_like(self.k[step]))
            write_kv_pages(k, self.v[step], self.keys, self.values, self.ks, self.vs, self.batch_table, before, self.row_starts,
                           max_query_len=ROWS)
            ancestors[:, :, step] = self.slots[step].view(REQS, ROWS).int()  # (row j of a step is a child of row j before it)
            out, n = torch.empty_like(q), REQS * HQ * 3 * 16
            part, lse = torch.empty(n, DIM, device=dev), torch.empty(n, device=dev)
            rows_attention(q, self.keys, self.values, out, part, lse, self.batch_table, self.context, ancestors, rows_per_request=ROWS,
                           step=step + 1, window=0, scale=DIM**-0.5, launch=RowsLaunch(splits=2, block_n=32), table_page=PAGE,
                           k_scale=self.ks, v_scale=self.vs)
            nodes = slice(step * REQS * ROWS, (step + 1) * REQS * ROWS)
            logits = 4 * out.reshape(REQS * ROWS, -1).float()[:, self.mix] + self.noise[nodes]
            probs = torch.empty(REQS * ROWS, VOCAB, device=dev)
            tokens = draw_tokens(logits, self.coins[step], self.t, self.top_k, self.top_p, entries=self.of_rows, probs=probs)
            # the step's rows drew the tokens of the nodes 1 + ROWS step ..; their parents' rows hold what they were drawn from
            at = torch.arange(REQS, device=dev)[:, None] * WIDTH + 1 + ROWS * step + torch.arange(ROWS, device=dev)[None]
            self.drafted[at.flatten()] = tokens
            parent = self.parents[1 + ROWS * step : 1 + ROWS * (step + 1)]
            self.probs[(torch.arange(REQS, device=dev)[:, None] * WIDTH + parent[None]).flatten()] = probs
            got["steps"].append(dict(q=q, k=k, positions=positions, ancestors=ancestors.clone(), out=out, logits=logits, tokens=tokens,
                                     probs=probs, keys=self.keys.clone(), values=self.values.clone(), ks=self.ks.clone(),
                                     vs=self.vs.clone(), slots=self.slots[step].clone()))
        cut = truncate_logits(self.target, self.t, self.top_k, self.top_p, entries=self.of_nodes)
        sampled, count = sample_tree(cut, self.drafted, self.node_starts, self.idx, self.store.parents, self.store, self.walk_coins,
                                     self.final, self.t, draft_probs=self.probs)
        accepted = self.context + count
        resize_tables(self.table, self.pages, self.idx, accepted, self.free, self.num_free, PAGE)
        got.update(cut=cut, sampled=sampled, count=count, pages=self.pages.clone(), left=self.num_free.clone(), free=self.free.clone())
        return got


def _round(dev, seed):
    from eagle_harness.vllm.rotary import rotary_frequencies
    from eagle_harness.vllm.verify_layout import TreeStore

    r = Round(dev, seed)
    r.frequencies, _ = rotary_frequencies(32, 1e6, device=dev)
    r.store = TreeStore(5, WIDTH, dev)
    r.store.parents[:] = torch.tensor(PARENTS, dtype=torch.int32, device=dev)
    return r


def test_a_round_step_by_step(dev):
    announce("sampled draft round, eager")
    r = _round(dev, 1)
    table, pages, stack = [[0] * MOST for _ in range(5)], [0] * 5, r.free.tolist()
    idx, lens = r.idx.tolist(), r.lens.tolist()
    got = r.run()
    torch.cuda.synchronize()
    ora_tables.resized(table, pages, idx, [n + ROWS * STEPS for n in lens], stack, 40, PAGE)
    assert got["grown"][1].tolist() == pages
    assert all(got["grown"][0][s, : pages[s]].tolist() == table[s][: pages[s]] for s in range(5))
    t, k, p = r.t.tolist(), r.top_k.tolist(), r.top_p.tolist()
    batch = torch.tensor([table[s] for s in idx], dtype=torch.int32)
    for step, x in enumerate(got["steps"]):
        assert x["slots"].tolist() == [ora_tables.slot_of(table, pages, s, n + step * ROWS + j, PAGE) for s, n in zip(idx, lens)
                                       for j in range(ROWS)]
        for name, of in (("q", r.q), ("k", r.k)):  # 16-bit rows: half a step of the value, and of the products' fp32 roundings
            want = ora_rotary.rotated(of[step].double().cpu().numpy(), x["positions"].cpu().numpy(), r.frequencies.cpu().numpy(), False, 1.0)
            size = np.abs(of[step].double().cpu().numpy()).max() * 2
            assert (np.abs(x[name].double().cpu().numpy() - want) <= 2.0**-8 * np.abs(want) + 2.0**-21 * size).all()
        wide = [x[c].cpu().float().double() * x[s].cpu().double()[:, None, :, None] for c, s in (("keys", "ks"), ("values", "vs"))]
        kw = dict(rows_per_request=ROWS, step=step + 1, window=0, scale=DIM**-0.5, table_page=PAGE)
        q, anc = x["q"].cpu().double(), x["ancestors"].cpu()
        want = ora_rows.rows_attention(q, wide[0], wide[1], batch, r.lens, anc, **kw)
        size = ora_rows.rows_attention(q, wide[0], wide[1].abs(), batch, r.lens, anc, **kw)
        assert ((x["out"].cpu().double() - want).abs() <= (2.0**-8 + 2.0**-16) * size + 2.0**-8 * want.abs()).all()
        logits, coins = x["logits"].cpu().numpy(), r.coins[step].cpu().numpy()
        for n in range(REQS * ROWS):
            b = n // ROWS
            order, mass = ora_sampling.kept_part(logits[n], t[b], k[b], p[b])
            assert int(x["tokens"][n]) == ora_sampling.drawn(order, mass, float(coins[n]))
            share = np.zeros(VOCAB)
            share[order] = mass / mass.sum()
            assert (np.abs(x["probs"][n].double().cpu().numpy() - share) <= 1.01 * 2.0**-24 * share + 2.0**-126).all()
    probs, drafted = r.probs.cpu().numpy(), r.drafted.cpu().numpy()
    for b in range(REQS):
        rows = slice(b * WIDTH, (b + 1) * WIDTH)
        want = np.full((WIDTH, VOCAB), -np.inf, dtype=np.float32)
        for j in range(WIDTH):
            line = r.target[b * WIDTH + j].cpu().numpy()
            order, _ = ora_sampling.kept_part(line, t[b], k[b], p[b])
            want[j, order] = line[order]
        assert np.array_equal(got["cut"][rows].cpu().numpy(), want)
        tokens, _ = ora_sampling.walk(want, drafted[rows], np.array(PARENTS), r.walk_coins[rows].cpu().numpy(), float(r.final[b]), t[b],
                                      probs[rows])
        assert got["sampled"][b, : int(got["count"][b])].tolist() == list(tokens)
    ora_tables.resized(table, pages, idx, [n + c for n, c in zip(lens, got["count"].tolist())], stack, 40, PAGE)
    assert got["pages"].tolist() == pages and got["free"][: len(stack)].tolist() == stack and got["left"].tolist() == [len(stack)]


def _flat(got):
    out = []
    for v in got.values():
        if isinstance(v, list):
            for x in v:
                out += _flat(x)
        else:
            out += list(v) if isinstance(v, tuple) else [v]
    return out


def test_a_round_captured(dev):
    """The same round replayed as one graph, each time from the state that the eager run starts with."""
    announce("sampled draft round, captured")
    r, state = _round(dev, 7), ("table", "pages", "free", "num_free", "keys", "values", "ks", "vs", "drafted", "probs")
    raw = lambda x: x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x  # noqa: E731
    first = {n: raw(getattr(r, n)).clone() for n in state}

    def back():
        for n in state:
            raw(getattr(r, n)).copy_(first[n])

    for _ in range(2):
        back()
        r.run()
    torch.cuda.synchronize()
    back()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = r.run()
    for seed in range(3):
        gen = torch.Generator().manual_seed(seed)
        lens = torch.randint(1, 60, (REQS,), generator=gen).int()
        r.context.copy_(lens)
        r.starts.copy_(torch.cat([torch.zeros(1), torch.cumsum(lens, 0)]).int())
        for x in (r.coins, r.walk_coins, r.final):
            x.copy_(torch.rand(x.shape, generator=gen))
        back()
        graph.replay()
        got = [raw(x).clone() for x in _flat(held)]
        back()
        want = [raw(x) for x in _flat(r.run())]
        torch.cuda.synchronize()
        counts = held["count"].tolist()
        assert all(1 <= c <= WIDTH for c in counts)
        for i, (a, b) in enumerate(zip(got, want)):
            if a.dtype == torch.int64 and a.shape == (REQS, WIDTH):  # sampled: -1 behind what was emitted
                assert torch.equal(a, b)
            else:
                assert torch.equal(a.view(torch.uint8) if a.is_floating_point() else a, b.view(torch.uint8) if b.is_floating_point() else b), i
