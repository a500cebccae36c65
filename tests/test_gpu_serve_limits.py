"""The serving operators where their numbers end: weights that are none, weights far
below a row's largest, scores and values that are not finite, sums that do not
come, rows in unusual places."""

import ctypes

import pytest
import torch

from tjkernels import _lib, ops
from tjkernels._lib import TjkError

from test_gpu_serve import U, Drafts, Trees, _half, _verify_oracle, _within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [37, 300, 50001])
@pytest.mark.parametrize("shape", ["chain", "tree"])
def test_negative_and_nan_draft_weights_are_zero(device, vocab, shape):
    """A token without any weight of the target's is not accepted because the draft's
    is negative, and gains none from it when others are refused."""
    for seed in range(6):
        d = Drafts([6, 9, 1, 12], vocab, shape, seed, noise=2.0)
        g = torch.Generator()
        g.manual_seed(seed)
        t = len(d.tokens)
        d.p[torch.rand(t, vocab, generator=g) < 0.5] = 0
        kind = torch.rand(t, vocab, generator=g)
        d.q[kind < 0.3] *= -1
        d.q[(kind > 0.3) & (kind < 0.4)] = float("nan")
        d.q[(kind > 0.4) & (kind < 0.45)] = -float("inf")
        # drafted tokens of each kind behind their parents
        d.tokens = torch.randint(0, vocab, (t,), generator=g).tolist()
        want = _verify_oracle(d.p, d.q.nan_to_num(0, neginf=0).clamp(min=0), d.tokens, d.parents, d.au, d.su, d.cu, d.n_max)
        assert d.run(device) == want


def _run_with_polls(d, device, polls):
    """d.run(device) where a workgroup looks `polls` times for another's sum."""
    call = _lib.load().tjk_verify_tree_polls
    types = _lib._SIGNATURES["tjk_verify_tree"][1]
    call.restype, call.argtypes = ctypes.c_int, types[:-1] + [ctypes.c_int] + types[-1:]
    batch, vocab, rows = len(d.counts), d.p.shape[1], len(d.tokens)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    need = _lib.load().tjk_verify_tree_bytes(vocab, batch)
    assert need > 0  # several workgroups
    workspace = torch.full((need,), 255, dtype=torch.uint8, device=device)
    path = torch.full((batch, d.n_max), 99, dtype=torch.int32, device=device)
    out = [path, i32([99] * batch), i32([99] * batch)]
    put = [x.to(device) for x in (d.p, d.q, d.au, d.su)] + [i32(d.tokens), i32(d.parents), i32(d.cu)]
    p, q, au, su, tokens, parents, cu = [x.data_ptr() for x in put]
    assert call(p, vocab, q, vocab, tokens, parents, au, su, cu, path.data_ptr(), d.n_max, out[1].data_ptr(), out[2].data_ptr(),
                None, rows, vocab, batch, d.n_max, workspace.data_ptr(), need, polls,
                torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    return tuple(x.tolist() for x in out)


@pytest.mark.parametrize("polls", [0, 1, 2, 5])
@pytest.mark.parametrize("counts,vocab", [([12, 20], 128257), ([64], 300001), ([9, 1, 0, 17] * 10, 50001)])
def test_verify_without_the_others_sums(device, polls, counts, vocab):
    """Workgroups that miss some or all of the others' sums compute them themselves:
    the same paths and tokens, with many refusals, without any, and where a residual is
    nothing."""
    assert _lib.load().tjk_verify_tree_bytes(vocab, len(counts)) > 0
    for seed in range(3):
        d = Drafts(counts, vocab, "tree", seed, noise=(1.0, 4.0, 0.1)[seed])
        if seed == 1:
            d.au = 1 - d.au / 8  # refusals
            b = counts[0]
            d.p[:b], d.q[:b] = 1 / (2 * vocab), 1 / vocab  # p below q everywhere
        assert _run_with_polls(d, device, polls) == d.want()
    d = Drafts([64] if len(counts) == 1 else [64, 3], vocab, "chain", 7, noise=3.0)
    d.parents = [-1] + [0] * 63 + ([] if len(counts) == 1 else [-1, 0, 0])  # 63 children of the root, most refused
    d.tokens[1:64] = (d.q[0] - d.p[0]).topk(63).indices.tolist()
    d.au[1:64] = 1 - 2.0 ** -20
    assert _run_with_polls(d, device, polls) == d.want()


def _set_scores(t, b, scores):
    """Keys of sequence b with these scores, for a scale of 1: the queries are the
    first unit vector."""
    x = torch.arange(len(scores))
    t.q.zero_()
    t.q[..., 0] = 1
    t.k[t.table[b][x // t.page].long(), 0, x % t.page, 0] = scores.to(t.dt)


@pytest.mark.parametrize("low,high", [(-18.2, -17.4), (-18.0, -9.7), (-22.0, -18.0)])
@pytest.mark.parametrize("sink", [0.0, 0.37, 1.0])
@pytest.mark.parametrize("nodes,heads,batch", [(1, 1, 600), (64, 2, 300)])
def test_far_smaller_weights_of_many_keys(device, low, high, sink, nodes, heads, batch):
    """One key takes most of a row, and 99995 others, 2^14 to 2^32 below it, give what
    its value, zero, leaves.  So many sequences share the pages that each is one
    workgroup's, and every key of a wave is held against the same offset.  fp16 weights
    are off by half a step, and by 2^-25 at least, where the largest is 2^7 or more: by
    2^-32 of it, in the weights' sum too."""
    n = 99995
    t = Trees([n - 1], [nodes], heads, 1, 16, 64, torch.float16, 40)
    t.mask[:] = 1  # the first node
    s = low + (high - low) * torch.rand(n, generator=t.g)
    s[int(sink * (n - 1))] = 0
    _set_scores(t, 0, s)
    t.v = (0.5 + 0.5 * torch.rand(t.v.shape, generator=t.g)).half()
    at = int(sink * (n - 1))
    t.v[t.table[0, at // 64], :, at % 64] = 0
    x = torch.arange(n)
    page, row = t.table[0][x // 64].long(), x % 64
    k, v = t.k[page, 0, row, 0].double(), t.v[page, 0, row].double()
    p = torch.softmax(k, 0)
    want = p @ v
    # (see Trees.exact: scores are exact here, the weights' arguments and sums are not)
    err = want * (2 * (((k.max() - k.min()) * 1.45 + 6) * U + _half(t.dt)) + 2 * (n + 8) * U) + 2 * 2.0 ** -32 * p.max() * v.sum(0)
    got = ops.tree_attention(t.q.repeat(batch, 1, 1).to(device), t.k.to(device), t.v.to(device),
                             t.table.repeat(batch, 1).to(device), t.ctx.repeat(batch).to(device),
                             torch.full((batch * nodes, heads * 16), 7.0, dtype=t.dt, device=device),
                             cu_nodes=torch.arange(0, batch * nodes + 1, nodes, dtype=torch.int32, device=device),
                             max_nodes=nodes, tree_mask=t.mask.repeat(batch).to(device), scale=1.0)
    _within(got.view(-1, 16), want, err, t.dt)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_scores_that_rise_along_a_row(device, dt):
    """Slowly, so that weights grow far past 1 before the row's offset follows: none
    passes the type's range."""
    for span in (5.5, 60.0, 700.0):
        t = Trees([3001, 40, 20000], [1, 1, 1], 2, 1, 16, 64, dt, 42, mask=None)
        for b, c in enumerate(t.contexts):
            _set_scores(t, b, torch.linspace(-span, 0, c + 1))
        t.check(device, scale=1.0)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("contexts,counts,heads,kv,hd", [([70, 0], [3, 5], 4, 2, 64), ([5000, 1], [1, 1], 1, 1, 64),
                                                         ([90, 200], [64, 40], 8, 2, 128)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_rows_of_infinitely_low_scores_are_zero(device, dt, contexts, counts, heads, kv, hd, bad):
    """Keys that take every row to -inf give a row of zeros, whatever their values
    hold."""
    t = Trees(contexts, counts, heads, kv, hd, 16, dt, 41)
    t.q = t.q.abs() + 1
    t.k[:] = -float("inf")
    t.v[:, :, ::3] = bad
    got = t.run(device)
    assert (got == 0).all()


def test_cache_of_steps_that_do_not_nest(device):
    """Heads between the rows of pages that lie closer than a page's heads reach: no
    two share a place, so the cache is as good as another."""
    t = Trees([11, 6], [3, 2], 6, 3, 16, 16, torch.bfloat16, 43)
    t.table = torch.tensor([[1], [0]], dtype=torch.int32)
    t.k, t.v, t.pages = t.k[:2].contiguous(), t.v[:2].contiguous(), 2
    want = t.run(device)
    odd = [torch.full((16 * 128,), 7.0, dtype=t.dt, device=device).as_strided((2, 3, 16, 16), (48, 32, 128, 1)) for _ in range(2)]
    # each position of the two sequences, appended
    x = torch.cat([torch.arange(14), torch.arange(8)])
    page = torch.tensor([1] * 14 + [0] * 8)
    rows = torch.cat([t.k[page, :, x], t.k[page, :, x], t.k[page, :, x], t.v[page, :, x]], dim=1).to(device)
    ops.rope_append(rows, x.int().to(device), None, torch.empty_like(rows[:, :6]), *odd, (page * 16 + x).int().to(device))
    assert torch.equal(t.run(device, k_cache=odd[0], v_cache=odd[1]), want)


def test_queries_and_output_in_one_buffer(device):
    """Side by side in its rows: the same bits; over each other: refused."""
    t = Trees([90, 33], [5, 12], 4, 2, 64, 16, torch.float16, 44)
    want = t.run(device)
    both = torch.full((t.t, 2, 256), 7.0, dtype=t.dt, device=device)
    both[:, 1] = t.q.view(t.t, 256).to(device)
    q = both[:, 1].unflatten(1, (4, 64))
    assert torch.equal(t.run(device, q=q, out=both[:, 0]), want)
    assert torch.equal(both[:, 1].cpu(), t.q.view(t.t, 256))
    with pytest.raises(TjkError, match="overlap"):
        t.run(device, q=q, out=both.view(-1)[248:].as_strided((t.t, 256), (512, 1)))
    k = t.k.to(device)
    args = [torch.zeros(3, dtype=torch.int32, device=device)] * 2
    qkv = torch.zeros(3, 8, 64, dtype=t.dt, device=device)
    with pytest.raises(TjkError, match="keys and values overlap"):
        ops.rope_append(qkv, args[0], None, torch.empty_like(qkv[:, :4]), k, k, args[1])
    with pytest.raises(TjkError, match="q_out and k_out overlap"):
        ops.rope_append(qkv, args[0], None, k.view(-1, 4, 64)[:3], k_out=k.view(-1, 2, 64)[1:4])


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("context", [2 ** 31 - 1, 2 ** 31 - 130])
def test_contexts_at_the_end_of_32_bits(device, dt, context):
    """A table of 2^31 positions, all of them rows of one page, and a context that
    reaches the last whole tile that 32 bits number, or past it: no row without a key is
    counted, which all of the keys, far below its score of zero, would vanish beside."""
    k = torch.zeros(1, 1, 65536, 16, dtype=dt, device=device)
    k[..., 0] = -100
    v = torch.ones_like(k)
    q = torch.zeros(1, 1, 16, dtype=dt, device=device)
    q[..., 0] = 1
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    errors = i32(0)
    out = torch.full((1, 16), 7.0, dtype=dt, device=device)
    ops.tree_attention(q, k, v, torch.zeros(1, 32768, dtype=torch.int32, device=device), i32(context), out, cu_nodes=i32(0, 1),
                       max_nodes=1, scale=1.0, index_errors=errors)
    assert (out == 1).all()
    assert int(errors) == (context + 1 > 2 ** 31 - 129)  # what is past it is cut off


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_append_keeps_the_bits_of_what_it_copies(device, dt):
    """Every number of the type, subnormals and infinities among them, as a value, and
    as a query and a key without norm and rotation; NaN stays NaN."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dt).view(512, 1, 128)
    qkv = bits.repeat(1, 3, 1).to(device)
    k, v = [torch.zeros(32, 1, 16, 128, dtype=dt, device=device) for _ in range(2)]
    at = torch.arange(512, dtype=torch.int32, device=device)
    q, k_out = torch.zeros_like(qkv[:, :1]), torch.zeros_like(qkv[:, :1])
    ops.rope_append(qkv, at, None, q, k, v, at, k_out=k_out)
    nan = torch.isnan(bits).flatten()
    want = bits.view(torch.int16).flatten()[~nan]
    for got in (q, k_out, k, v):
        got = got.cpu().flatten()
        assert torch.isnan(got[nan]).all() and torch.equal(got.view(torch.int16)[~nan], want)
