"""The serving operators together, as a program uses them: a model's prompt and
steps of drafted tokens, graphs, two calls at once."""

import pytest
import torch

from tjkernels import _lib, ops
from tjkernels.graphs import CapturedGraph

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


class Server:
    """Layers of attention alone (projections would only add noise): every
    token's packed qkv is given, per layer."""

    def __init__(self, device, layers, batch, heads, hd, page, per_seq, dt):
        self.device, self.layers, self.heads, self.hd, self.page, self.dt = device, layers, heads, hd, page, dt
        pages = batch * per_seq
        self.k = torch.zeros(layers, pages, heads, page, hd, dtype=dt, device=device)
        self.v = torch.zeros_like(self.k)
        self.table = torch.randperm(pages, generator=_gen(1)).int().view(batch, per_seq).to(device)
        self.ctx = torch.zeros(batch, dtype=torch.int32, device=device)
        self.angles = ops.rope_table(per_seq * page, hd, device=device)

    def slots(self, b, x):
        x = x.to(self.device)
        return (self.table[b.to(self.device), (x // self.page).long()] * self.page + x % self.page).int()

    def prompt(self, qkv, lengths):
        """Causal attention of packed prompts, their keys and values stored."""
        h, hd, t = self.heads, self.hd, sum(lengths)
        b = torch.cat([torch.full((n,), i) for i, n in enumerate(lengths)])
        pos = torch.cat([torch.arange(n) for n in lengths]).int()
        cu = torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32, device=self.device)
        outs = []
        for layer in range(self.layers):
            x = qkv[layer].clone()
            flat = x.view(t, 3 * h, hd)
            ops.rope_append(flat, pos.to(self.device), self.angles, flat[:, :h], self.k[layer], self.v[layer],
                            self.slots(b, pos), k_out=flat[:, h:2 * h])
            out = torch.empty(t, h * hd, dtype=self.dt, device=self.device)
            ops.flash_attention(x.view(t, 3, h, hd), out, cu_seqlens=cu, max_seqlen=max(lengths))
            outs.append(out)
        self.ctx += torch.tensor(lengths, dtype=torch.int32, device=self.device)
        return outs

    def step(self, qkv, counts, depth, mask):
        """One step of trees (rows back to back), behind what is stored."""
        h, hd = self.heads, self.hd
        cu = torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device=self.device)
        b = torch.cat([torch.full((n,), i) for i, n in enumerate(counts)])
        node = torch.cat([torch.arange(n) for n in counts]).int()
        ctx = self.ctx[b.to(self.device)]
        slots = self.slots(b, ctx.cpu() + node)
        outs = []
        for layer in range(self.layers):
            flat = qkv[layer].view(-1, 3 * h, hd)
            q = torch.empty(flat.shape[0], h, hd, dtype=self.dt, device=self.device)
            ops.rope_append(flat, ctx + depth, self.angles, q, self.k[layer], self.v[layer], slots)
            out = torch.empty(flat.shape[0], h * hd, dtype=self.dt, device=self.device)
            ops.tree_attention(q, self.k[layer], self.v[layer], self.table, self.ctx, out, cu_nodes=cu,
                               max_nodes=max(counts), tree_mask=mask)
            outs.append(out)
        return outs


def _close(got, want, dt):
    """Two kernels on the same rounded queries, keys and values: each rounds its
    weights and its result once, half a step of values of size 5 at most (the
    context of standard normal values), with fp32 sums far below that."""
    step = torch.finfo(dt).eps / 2
    diff = (got.float() - want.float()).abs()
    assert (diff <= 4 * step * 5).all(), float(diff.max())


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,hd,page", [(4, 64, 16), (2, 128, 64)])
def test_prompt_then_single_tokens(device, dt, heads, hd, page):
    """Token by token over the cache is what causal attention over the whole
    sequence gives."""
    g, layers, lengths, more = _gen(3), 2, [37, 5, 64], 6
    whole = torch.randn(layers, sum(lengths) + 3 * more, 3, heads, hd, generator=g).to(dt).to(device)
    rows = [[], []]  # rows of the prompts, and of the tokens behind them, by sequence
    at = 0
    for n in lengths:
        rows[0].append(list(range(at, at + n)))
        rows[1].append(list(range(at + n, at + n + more)))
        at += n + more
    want = Server(device, layers, 3, heads, hd, page, 128 // page, dt).prompt(whole, [n + more for n in lengths])
    s = Server(device, layers, 3, heads, hd, page, 128 // page, dt)
    first = sum(rows[0], [])
    got = s.prompt(whole[:, first].contiguous(), lengths)
    for layer in range(layers):
        _close(got[layer], want[layer][first], dt)
    zero = torch.zeros(3, dtype=torch.int32, device=device)
    for i in range(more):
        now = [r[i] for r in rows[1]]
        got = s.step(whole[:, now].contiguous(), [1, 1, 1], zero, None)
        s.ctx += 1
        for layer in range(layers):
            _close(got[layer], want[layer][now], dt)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_steps_of_drafted_trees(device, dt):
    """Append, attend, verify, compact: a node's attention is that of its path
    written out as a sequence, and after the accepted path is compacted the
    cache holds what the kept tokens alone would have left."""
    g, layers, heads, hd, page, vocab = _gen(5), 2, 4, 64, 16, 97
    lengths = [20, 47]
    s = Server(device, layers, 2, heads, hd, page, 8, dt)
    prompts = torch.randn(layers, sum(lengths), 3, heads, hd, generator=g).to(dt).to(device)
    s.prompt(prompts, lengths)
    kept = [[prompts[:, :20]], [prompts[:, 20:]]]
    parents = [-1, 0, 0, 1, 1, 2, 3, 3, 5]
    depth, bits = [0], [1]
    for j in range(1, 9):
        depth.append(depth[parents[j]] + 1)
        bits.append(bits[parents[j]] | 1 << j)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    longest = 0
    for _ in range(4):
        rows = torch.randn(layers, 18, 3, heads, hd, generator=g).to(dt).to(device)
        out = s.step(rows, [9, 9], i32(depth * 2), torch.tensor(bits * 2, device=device))
        logits = torch.randn(18, vocab, generator=g)
        p = torch.softmax(logits, 1)
        q = torch.softmax(logits + 0.2 * torch.randn(18, vocab, generator=g), 1)
        tokens = [int(torch.multinomial(q[9 * b + max(parents[j], 0)], 1, generator=g)) for b in range(2) for j in range(9)]
        path, count, token = torch.empty(2, 9, dtype=torch.int32, device=device), i32([0, 0]), i32([0, 0])
        ops.verify_tree(p.to(device), q.to(device), i32(tokens), i32(parents * 2), torch.rand(18, generator=g).to(device),
                        torch.rand(2, generator=g).to(device), path, count, token, cu_nodes=i32([0, 9, 18]))
        ops.compact_cache(s.k, s.v, s.table, s.ctx, path, count)
        s.ctx += count
        longest = max(longest, int(count.max()))
        for b in range(2):
            taken = path[b, :int(count[b])].tolist()
            kept[b].append(rows[:, [9 * b + j for j in taken]])
            # the accepted path as a plain sequence, with causal attention
            plain = Server(device, layers, 1, heads, hd, page, 8, dt)
            seq = torch.cat(kept[b], dim=1).contiguous()
            want = plain.prompt(seq, [seq.shape[1]])
            n = seq.shape[1]
            x = torch.arange(n)
            mine, its = s.slots(torch.full((n,), b), x).long(), plain.slots(torch.zeros(n, dtype=torch.long), x).long()
            for layer in range(layers):
                _close(out[layer][[9 * b + j for j in taken]], want[layer][n - len(taken):], dt)
                for a, c in ((s.k, plain.k), (s.v, plain.v)):
                    assert torch.equal(a[layer][mine // page, :, mine % page], c[layer][its // page, :, its % page])
    assert longest > 2


def _inputs(device, seed, dt=torch.bfloat16, context=(1500, 40)):
    g = _gen(seed)
    heads, kv, hd, page, counts, vocab = 8, 2, 64, 32, [5, 9], 1000
    table = torch.randperm(120, generator=g).int().view(2, 60)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    ctx = i32(list(context))
    node = i32([0, 1, 2, 3, 4] + list(range(9)))
    b = torch.tensor([0] * 5 + [1] * 9)
    x = ctx[b] + node
    logits = torch.randn(14, vocab, generator=g)
    d = dict(qkv=torch.randn(14, heads + 2 * kv, hd, generator=g).to(dt), pos=x, table=ops.rope_table(2048, hd),
             slots=table[b, (x // page).long()] * page + x % page, k=torch.randn(2, 120, kv, page, hd, generator=g).to(dt),
             v=torch.randn(2, 120, kv, page, hd, generator=g).to(dt), blocks=table, ctx=ctx, cu=i32([0, 5, 14]),
             p=torch.softmax(logits, 1), qd=torch.softmax(logits + torch.randn(14, vocab, generator=g), 1),
             tokens=torch.randint(0, vocab, (14,), generator=g).int(), parents=i32([-1, 0, 0, 1, 2, -1, 0, 0, 1, 1, 2, 3, 3, 4]),
             au=torch.rand(14, generator=g), su=torch.rand(2, generator=g))
    d = {k: v.to(device) for k, v in d.items()}
    d.update(q=torch.empty(14, heads, hd, dtype=dt, device=device), out=torch.empty(14, heads * hd, dtype=dt, device=device),
             path=torch.empty(2, 9, dtype=torch.int32, device=device), count=torch.empty(2, dtype=torch.int32, device=device),
             token=torch.empty(2, dtype=torch.int32, device=device))
    return d


def _step(d, ws=None):
    for layer in range(2):
        ops.rope_append(d["qkv"], d["pos"], d["table"], d["q"], d["k"][layer], d["v"][layer], d["slots"])
        ops.tree_attention(d["q"], d["k"][layer], d["v"][layer], d["blocks"], d["ctx"], d["out"], cu_nodes=d["cu"], max_nodes=9,
                           workspace=ws)
    ops.verify_tree(d["p"], d["qd"], d["tokens"], d["parents"], d["au"], d["su"], d["path"], d["count"], d["token"],
                    cu_nodes=d["cu"])
    ops.compact_cache(d["k"], d["v"], d["blocks"], d["ctx"], d["path"], d["count"])


OUT = ("q", "out", "path", "count", "token", "k", "v")


def test_step_captured_beside_a_graph_of_inference_mode(device):
    """The engine's callers are under inference_mode, and so are its captures; while
    such a graph lives, a step can be captured outside of it, and in it."""
    x = torch.ones(4, device=device)
    with torch.inference_mode():
        kept = CapturedGraph(lambda: x.add_(1), device)
    d = _inputs(device, 1)
    _step(d)
    for mode in (False, True):
        with torch.inference_mode(mode):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                ops.tree_attention(d["q"], d["k"][0], d["v"][0], d["blocks"], d["ctx"], d["out"], cu_nodes=d["cu"], max_nodes=9)
        want = ops.tree_attention(d["q"], d["k"][0], d["v"][0], d["blocks"], d["ctx"], torch.empty_like(d["out"]),
                                  cu_nodes=d["cu"], max_nodes=9)
        d["out"].zero_()
        graph.replay()
        assert torch.equal(d["out"], want)
    kept.replay()
    assert (x == 3).all()


@pytest.mark.parametrize("own_workspace", [True, False])
def test_captured_step(device, own_workspace):
    """A whole step in a graph, replayed on new inputs and other lengths, with
    eager steps in between."""
    d = _inputs(device, 1)
    ws = ops.tree_attention_workspace(d["q"], d["k"][0], 9) if own_workspace else None
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(d, ws)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _step(d, ws)
    for seed, context in ((2, (1500, 40)), (3, (10, 1900)), (4, (0, 0)), (5, (1911, 7))):
        new = _inputs(device, seed, context=context)
        for k in d:
            d[k].copy_(new[k])
        graph.replay()
        _step(new)
        torch.cuda.synchronize()
        for k in OUT:
            assert torch.equal(d[k], new[k]), (seed, k)


def test_two_graphs_share_a_workspace(device):
    """Captured apart, replayed in turn on one stream."""
    ds = [_inputs(device, 7), _inputs(device, 8, context=(3, 1700))]
    ws = ops.tree_attention_workspace(ds[0]["q"], ds[0]["k"][0], 9)
    graphs = []
    for d in ds:
        _step({**d, "k": d["k"].clone(), "v": d["v"].clone()}, ws)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _step(d, ws)
        graphs.append(graph)
    for _ in range(3):
        for d, graph, seed, context in zip(ds, graphs, (7, 8), ((1500, 40), (3, 1700))):
            new = _inputs(device, seed, context=context)
            for k in ("k", "v"):
                d[k].copy_(new[k])
            d["out"].zero_()
            graph.replay()
            _step(new)
            for k in OUT:
                assert torch.equal(d[k], new[k]), k


def test_two_calls_at_once(device):
    """Steps on two streams, each with its own workspace, overlap as they like."""
    jobs = [_inputs(device, 11, context=(1800, 1700)), _inputs(device, 12, context=(1600, 1900))]
    wants = [_inputs(device, 11, context=(1800, 1700)), _inputs(device, 12, context=(1600, 1900))]
    for d in wants:
        _step(d)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    works = [ops.tree_attention_workspace(d["q"], d["k"][0], 9) for d in jobs]
    torch.cuda.synchronize()
    for _ in range(5):
        for d, stream, ws in zip(jobs, streams, works):
            with torch.cuda.stream(stream):
                ops.rope_append(d["qkv"], d["pos"], d["table"], d["q"], d["k"][1], d["v"][1], d["slots"])
                ops.tree_attention(d["q"], d["k"][1], d["v"][1], d["blocks"], d["ctx"], d["out"], cu_nodes=d["cu"],
                                   max_nodes=9, workspace=ws)
                ops.verify_tree(d["p"], d["qd"], d["tokens"], d["parents"], d["au"], d["su"], d["path"], d["count"],
                                d["token"], cu_nodes=d["cu"])
    torch.cuda.synchronize()
    for d, want in zip(jobs, wants):
        for k in ("q", "out", "path", "count", "token"):
            assert torch.equal(d[k], want[k]), k


def _verification(device, seed, batch=3, vocab=150001):
    """Arguments of a verification that several workgroups share."""
    g = _gen(seed)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    logits = torch.randn(5 * batch, vocab, generator=g)
    a = [torch.softmax(logits, 1), torch.softmax(logits + 2 * torch.randn(5 * batch, vocab, generator=g), 1),
         torch.randint(0, vocab, (5 * batch,), generator=g).int(), i32([-1, 0, 0, 0, 1] * batch),
         torch.rand(5 * batch, generator=g), torch.rand(batch, generator=g)]
    a[2][1::5] = a[0][0::5].argmax(1).int()
    return [x.to(device) for x in a], i32([5 * b for b in range(batch + 1)]).to(device)


def _verified(device, a, cu, workspace=None):
    batch = cu.numel() - 1
    path = torch.zeros(batch, 5, dtype=torch.int32, device=device)
    count, token = torch.zeros_like(path[:, 0]).contiguous(), torch.zeros_like(path[:, 0]).contiguous()
    ops.verify_tree(*a, path, count, token, cu_nodes=cu, workspace=workspace)
    return path, count, token


@pytest.mark.parametrize("own_workspace", [True, False])
def test_captured_verification_of_several_workgroups(device, own_workspace):
    """Replayed on other distributions and numbers, with eager calls in between."""
    a, cu = _verification(device, 1)
    need = _lib.load().tjk_verify_tree_bytes(150001, 3)
    assert need > 0
    ws = torch.full((need,), 255, dtype=torch.uint8, device=device) if own_workspace else None
    _verified(device, a, cu, ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _verified(device, a, cu, ws)
    seen = set()
    for seed in range(2, 7):
        new, _ = _verification(device, seed)
        for x, y in zip(a, new):
            x.copy_(y)
        graph.replay()
        want = _verified(device, new, cu)
        torch.cuda.synchronize()
        for x, y in zip(out, want):
            assert torch.equal(x, y), seed
        seen |= set(want[2].tolist())
    assert len(seen) > 10


def test_verifications_at_once(device):
    """Two streams' verifications share the chip, beside attention over long
    contexts that may hold its workgroups up: the same results."""
    jobs = [_verification(device, seed, batch, vocab) for seed, batch, vocab in ((21, 3, 150001), (22, 16, 60001))]
    wants = [_verified(device, *job) for job in jobs]
    d = _inputs(device, 23, context=(1800, 1700))
    want = torch.empty_like(d["out"])
    attend = lambda out: ops.tree_attention(d["q"], d["k"][0], d["v"][0], d["blocks"], d["ctx"], out, cu_nodes=d["cu"],  # noqa: E731
                                            max_nodes=9)
    d["q"].normal_()
    attend(want)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for _ in range(8):
        for job, stream in zip(jobs, streams):
            with torch.cuda.stream(stream):
                got.append(_verified(device, *job))
        with torch.cuda.stream(streams[2]):
            attend(d["out"])
    torch.cuda.synchronize()
    for i, result in enumerate(got):
        for x, y in zip(result, wants[i % 2]):
            assert torch.equal(x, y)
    assert torch.equal(d["out"], want)
