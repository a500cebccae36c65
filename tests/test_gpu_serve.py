"""The serving operators against 64-bit results of the same inputs: the rotated
append to a paged cache, attention of drafted trees over it, verification and
compaction.  Tolerances are bounds on the kernels' own roundings, derived beside
each."""

import pytest
import torch

from tjkernels import ops

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24  # half a unit in the last place of fp32, relative
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # half the least number of a type


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _half(dt):
    return torch.finfo(dt).eps / 2


def _within(got, want, err, dt):
    """got (of type dt) is want, known to within err, rounded to dt."""
    got = got.double().cpu()
    bound = err + _half(dt) * (want.abs() + err) + TINY[dt]
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst by {((got - want).abs() / bound).max():.3g} bounds"


# ------------------------------------------------------------------- append

def _rotate(x, cs, interleaved):
    """64-bit x [T, rows, hd], cs [T, half, 2]: rotated, and the size of the
    terms that were added."""
    half = cs.shape[1]
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    y, size = x.clone(), x.abs()
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    size[..., a] = (x[..., a] * c).abs() + (x[..., b] * s).abs()
    size[..., b] = (x[..., b] * c).abs() + (x[..., a] * s).abs()
    return y, size


def _append_case(t, heads, kv, hd, rot, norms, interleaved, dt, seed):
    g = _gen(seed)
    qkv = (torch.randn(t, heads + 2 * kv, hd, generator=g) * torch.exp(torch.randn(t, 1, 1, generator=g))).to(dt)
    table = ops.rope_table(1000, rot)
    pos = torch.randint(0, 1000, (t,), generator=g).int()
    qg, kg = (1 + 0.2 * torch.randn(hd, generator=g), 1 + 0.2 * torch.randn(hd, generator=g)) if norms else (None, None)
    x = qkv.double()
    rows = heads + kv
    if norms:
        r = 1 / (x[:, :rows].square().mean(dim=2, keepdim=True) + 1e-6).sqrt()
        x = torch.cat([x[:, :heads] * r[:, :heads] * qg.double(), x[:, heads:rows] * r[:, heads:] * kg.double(), x[:, rows:]],
                      dim=1)
    y, size = _rotate(x[:, :rows], table[pos.long()].double(), interleaved)
    # the sum of squares, its root and the two products of the norm; three
    # roundings of the rotation
    err = size * U * ((hd / 8 + 12 if norms else 0) + 3)
    return qkv, table, pos, qg, kg, y, err


APPEND = [
    # t, heads, kv, hd, rot, norms, interleaved, page
    (1, 1, 1, 16, 16, True, False, 16), (3, 2, 1, 32, 16, False, True, 16), (7, 3, 3, 48, 32, True, False, 32),
    (33, 8, 2, 64, 64, True, False, 16), (130, 16, 16, 64, 64, False, True, 64), (5, 12, 4, 80, 80, True, True, 16),
    (17, 6, 3, 96, 48, True, False, 32), (9, 4, 4, 112, 112, False, False, 16), (64, 32, 8, 128, 128, True, False, 128),
    (257, 5, 1, 128, 64, True, True, 16), (11, 16, 2, 128, 0, True, False, 16), (4, 40, 40, 128, 128, False, False, 256),
]


@pytest.mark.parametrize("t,heads,kv,hd,rot,norms,interleaved,page", APPEND)
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_append(device, t, heads, kv, hd, rot, norms, interleaved, page, dt):
    """Queries, keys and values land where they belong, every other element of
    the outputs and of a cache with padded rows stays."""
    dt = DT[dt]
    qkv, table, pos, qg, kg, y, err = _append_case(t, heads, kv, hd, rot, norms, interleaved, dt, t * hd)
    pages = -(-t // page) + 2
    slots = torch.randperm(pages * page, generator=_gen(t))[:t].int()
    slots[::5] = -1 - (slots[::5] % 3)
    k_whole = torch.full((pages, kv, page, hd + 8), 7.0, dtype=dt, device=device)
    v_whole = torch.full((pages, kv, page, hd + 8), 7.0, dtype=dt, device=device)
    q_whole = torch.full((t + 2, heads, hd + 16), 7.0, dtype=dt, device=device)
    k_out = torch.full((t, kv, hd), 7.0, dtype=dt, device=device)
    put = lambda x: None if x is None else x.to(device)  # noqa: E731
    errors = torch.zeros(1, dtype=torch.int32, device=device)
    ops.rope_append(put(qkv), put(pos), put(table) if rot else None, q_whole[1:t + 1, :, :hd], k_whole[..., :hd],
                    v_whole[..., :hd], put(slots), k_out=k_out, q_gamma=put(qg), k_gamma=put(kg), interleaved=interleaved,
                    index_errors=errors)
    _within(q_whole[1:t + 1, :, :hd], y[:, :heads], err[:, :heads], dt)
    _within(k_out, y[:, heads:], err[:, heads:], dt)
    assert int(errors) == 0
    kept = slots >= 0
    at = slots[kept].long()
    k_got, v_got = k_whole.cpu(), v_whole.cpu()
    assert torch.equal(k_got[at // page, :, at % page, :hd], k_out.cpu()[kept])
    assert torch.equal(v_got[at // page, :, at % page, :hd], qkv[kept][:, heads + kv:])
    k_got[at // page, :, at % page, :hd] = 7
    v_got[at // page, :, at % page, :hd] = 7
    q_whole[1:t + 1, :, :hd] = 7
    assert (k_got == 7).all() and (v_got == 7).all() and (q_whole == 7).all()


@pytest.mark.parametrize("hd,rot,interleaved", [(64, 64, False), (128, 64, True), (80, 80, False)])
def test_append_in_place_without_cache(device, hd, rot, interleaved):
    """A packed [T, 3, H, hd] buffer rotated in place is what the attention
    kernels read; its values stay."""
    t, heads = 37, 4
    qkv, table, pos, qg, kg, y, err = _append_case(t, heads, heads, hd, rot, True, interleaved, torch.bfloat16, 3)
    packed = qkv.to(device).clone()
    ops.rope_append(packed, pos.to(device), table.to(device), packed[:, :heads], k_out=packed[:, heads:2 * heads],
                    q_gamma=qg.to(device), k_gamma=kg.to(device), interleaved=interleaved)
    _within(packed[:, :2 * heads], y, err, torch.bfloat16)
    assert torch.equal(packed[:, 2 * heads:].cpu(), qkv[:, 2 * heads:])


@pytest.mark.parametrize("t,heads", [(1, 4), (37, 1), (1, 1)])
def test_append_in_place_of_one(device, t, heads):
    """One token, one head: their views' strides say nothing, the rows are the
    same."""
    hd = 64
    qkv, table, pos, qg, kg, y, err = _append_case(t, heads, heads, hd, hd, True, False, torch.bfloat16, 13)
    padded = torch.full((t, 3 * heads, 72), 7.0, dtype=torch.bfloat16, device=device)
    padded[..., :hd] = qkv.to(device)
    rows = padded[..., :hd]
    ops.rope_append(rows, pos.to(device), table.to(device), rows[:, :heads], k_out=rows[:, heads:2 * heads],
                    q_gamma=qg.to(device), k_gamma=kg.to(device))
    _within(rows[:, :2 * heads], y, err, torch.bfloat16)
    assert torch.equal(rows[:, 2 * heads:].cpu(), qkv[:, 2 * heads:]) and (padded[..., hd:] == 7).all()


def test_append_cache_orders(device):
    """[pages, page, heads, hd] seen as [pages, heads, page, hd], keys and values
    side by side in one buffer, a strided qkv: the same rows."""
    t, heads, kv, hd, page = 21, 4, 2, 64, 16
    qkv, table, pos, qg, kg, _, _ = _append_case(t, heads, kv, hd, hd, True, False, torch.float16, 5)
    slots = torch.randperm(4 * page, generator=_gen(1))[:t].int().to(device)
    got = []
    both = torch.zeros(4, 2, page, kv, hd, dtype=torch.float16, device=device)
    plain = torch.zeros(2, 4, kv, page, hd, dtype=torch.float16, device=device)
    spread = torch.zeros(t, 2 * (heads + 2 * kv), hd, dtype=torch.float16, device=device)
    spread[:, ::2] = qkv.to(device)
    for src, k, v in ((qkv.to(device), plain[0], plain[1]),
                      (spread[:, ::2], both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2))):
        q = torch.empty(t, heads, hd, dtype=torch.float16, device=device)
        ops.rope_append(src, pos.to(device), table.to(device), q, k, v, slots, q_gamma=qg.to(device), k_gamma=kg.to(device))
        got.append((q, k.clone(), v.clone()))
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_append_bad_indexes(device):
    """Positions outside the table: zero rows, nothing stored, counted; slots
    outside the cache: nothing stored, counted; the others as ever."""
    t, heads, kv, hd, page = 8, 2, 1, 64, 16
    qkv, table, pos, _, _, y, err = _append_case(t, heads, kv, hd, hd, False, False, torch.bfloat16, 9)
    pos[1], pos[2], pos[5] = -1, 1000, 2 ** 31 - 1
    slots = torch.tensor([0, 1, 2, 3 * page, 4, 5, 2 ** 31 - 1, 7], dtype=torch.int32)
    k = torch.full((3, kv, page, hd), 7.0, dtype=torch.bfloat16, device=device)
    v, q = k.clone(), torch.full((t, heads, hd), 7.0, dtype=torch.bfloat16, device=device)
    k_out = torch.full((t, kv, hd), 7.0, dtype=torch.bfloat16, device=device)
    errors = torch.full((1,), 10, dtype=torch.int32, device=device)
    ops.rope_append(qkv.to(device), pos.to(device), table.to(device), q, k, v, slots.to(device), k_out=k_out,
                    index_errors=errors)
    assert int(errors) == 15
    lost = [1, 2, 5]
    assert (q[lost] == 0).all() and (k_out[lost] == 0).all()
    fine = [0, 3, 4, 6, 7]
    _within(q[fine], y[fine][:, :heads], err[fine][:, :heads], torch.bfloat16)
    stored = k[0, 0, [0, 4, 7]]
    assert torch.equal(stored, k_out[[0, 4, 7], 0])
    k[0, 0, [0, 4, 7]] = 7
    assert (k == 7).all()


# ---------------------------------------------------------------- attention

class Trees:
    """A batch over a paged cache, on the host in its own type."""

    def __init__(self, contexts, counts, heads, kv, hd, page, dt, seed, mask="tree", spread=1.0):
        g = self.g = _gen(seed)
        self.contexts, self.counts, self.heads, self.kv, self.hd, self.page, self.dt = \
            contexts, counts, heads, kv, hd, page, dt
        rows = [-(-(c + n) // page) for c, n in zip(contexts, counts)]
        self.pages = sum(rows) + 1
        order = (torch.randperm(self.pages - 1, generator=g) + 1).int()  # page 0 belongs to nobody
        self.table = torch.full((len(counts), max(rows + [1])), -1, dtype=torch.int32)
        at = 0
        for b, r in enumerate(rows):
            self.table[b, :r] = order[at:at + r]
            at += r
        self.k = torch.randn(self.pages, kv, page, hd, generator=g).to(dt)
        self.v = torch.randn(self.pages, kv, page, hd, generator=g).to(dt)
        self.t = sum(counts)
        self.q = (spread * torch.randn(self.t, heads, hd, generator=g)).to(dt)
        self.cu = torch.tensor([sum(counts[:b]) for b in range(len(counts) + 1)], dtype=torch.int32)
        self.ctx = torch.tensor(contexts, dtype=torch.int32)
        self.mask = None
        if mask == "tree":
            bits = []
            for n in counts:
                tree = []
                for j in range(n):
                    up = tree[int(torch.randint(0, j, (1,), generator=g))] if j else 0
                    tree.append(up | 1 << j)
                bits += tree
            self.mask = torch.tensor([b - (1 << 64) if b >> 63 else b for b in bits], dtype=torch.int64)
        self.max_nodes = max(counts + [1])

    def seen(self, b, i):
        """[context + n] truth values of node i of sequence b."""
        n, c = self.counts[b], self.contexts[b]
        bits = int(self.mask[self.cu[b] + i]) if self.mask is not None else (1 << i + 1) - 1
        keep = torch.ones(c + n, dtype=torch.bool)
        keep[c:] = torch.tensor([bool(bits >> j & 1) for j in range(n)], dtype=torch.bool)
        x = torch.arange(c + n)
        pages = self.table[b][(x // self.page).clamp(max=self.table.shape[1] - 1)]
        return keep & (x // self.page < self.table.shape[1]) & (pages >= 0) & (pages < self.pages)

    def exact(self, scale=None):
        """(out, error) [T, heads * hd] in 64 bits.

        Per row: a score is off by (hd + 2) U of its terms' sum (fp32 sums of
        exact products, the scale), its weight by that, by U times its exponent
        (an argument of up to `span` in base 2, rounded) and 2 units of exp2, and
        by the rounding of the weight to the type; the sums over n keys in fp32
        add n U at most.  The denominator's weights are off alike.  fp16 weights
        below 2^-14 of the largest are off by 2^-25 of it, absolute."""
        scale = self.hd ** -0.5 if scale is None else scale
        out = torch.zeros(self.t, self.heads, self.hd, dtype=torch.float64)
        err = torch.zeros_like(out)
        for b, (n, c) in enumerate(zip(self.counts, self.contexts)):
            x = torch.arange(c + n)
            for i in range(n):
                x_i = x[self.seen(b, i)]
                if x_i.numel() == 0:
                    continue
                page, row = self.table[b][x_i // self.page].long(), x_i % self.page
                k, v = self.k[page, :, row].double(), self.v[page, :, row].double()  # [keys, kv, hd]
                q = self.q[self.cu[b] + i].double().view(self.kv, -1, self.hd)
                terms = q.transpose(0, 1)[:, None] * k  # [group, keys, kv, hd]
                s = terms.sum(3) * scale
                ds = (self.hd + 2) * U * (terms.abs().sum(3) * abs(scale)).amax(1, keepdim=True)
                p = torch.softmax(s, dim=1)
                span = (s.amax(1, keepdim=True) - s.amin(1, keepdim=True)) * 1.45
                rel = 2 * (ds + (span + 6) * U + _half(self.dt)) + 2 * (x_i.numel() + 8) * U
                o = (p[..., None] * v).sum(1)
                size = (p[..., None] * v.abs()).sum(1)
                floor = 2.0 ** -25 * p.amax(1)[..., None] * v.abs().sum(0) * 2 if self.dt == torch.float16 else 0
                at = (slice(None),)
                out[self.cu[b] + i] = o.transpose(0, 1).reshape(self.heads, self.hd)
                err[self.cu[b] + i] = (rel.squeeze(1)[..., None] * size + floor).transpose(0, 1).reshape(self.heads, self.hd)[at]
        return out.view(self.t, -1), err.view(self.t, -1)

    def run(self, device, fill=7.0, rows=None, errors=None, **kw):
        put = lambda x: None if x is None else x.to(device)  # noqa: E731
        rows = self.t if rows is None else rows
        out = torch.full((rows, self.heads * self.hd), fill, dtype=self.dt, device=device)
        args = dict(q=put(self.q), k_cache=put(self.k), v_cache=put(self.v), block_table=put(self.table), ctx_lens=put(self.ctx),
                    out=out, cu_nodes=put(self.cu), max_nodes=self.max_nodes, tree_mask=put(self.mask), index_errors=errors)
        args.update(kw)
        return ops.tree_attention(**args)

    def check(self, device, scale=None, **kw):
        errors = torch.zeros(1, dtype=torch.int32, device=device)
        got = self.run(device, errors=errors, **({} if scale is None else dict(scale=scale)), **kw)
        want, err = self.exact(scale)
        _within(got, want, err, self.dt)
        assert int(errors) == 0
        return got


ATTEND = [
    # contexts, counts, heads, kv, hd, page
    ([0], [1], 1, 1, 16, 16), ([1], [1], 2, 1, 64, 16), ([31, 32, 33], [1, 1, 1], 4, 4, 64, 32),
    ([100, 0, 257, 64], [1, 1, 1, 1], 8, 8, 128, 16), ([15, 16, 17, 500], [1, 2, 3, 5], 6, 2, 48, 16),
    ([511, 90], [64, 33], 2, 2, 64, 64), ([63, 128, 1], [17, 64, 8], 16, 2, 32, 16), ([200, 70], [9, 5], 12, 4, 80, 32),
    ([300], [31], 8, 1, 96, 16), ([129, 40], [64, 50], 16, 2, 128, 32), ([600, 3], [7, 1], 3, 3, 112, 256),
    ([1000, 5, 333], [1, 1, 1], 32, 2, 128, 64), ([77, 200], [64, 64], 16, 1, 64, 16),
]


@pytest.mark.parametrize("contexts,counts,heads,kv,hd,page", ATTEND)
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("mask", ["tree", "chain"])
def test_attention(device, contexts, counts, heads, kv, hd, page, dt, mask):
    Trees(contexts, counts, heads, kv, hd, page, DT[dt], sum(contexts) + hd, mask).check(device)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("contexts,counts,heads,kv,hd", [([4100], [1], 2, 1, 64), ([2500, 3], [3, 2], 4, 2, 128),
                                                         ([9000], [12], 2, 2, 32)])
def test_long_contexts(device, contexts, counts, heads, kv, hd, dt):
    Trees(contexts, counts, heads, kv, hd, 64, DT[dt], 1).check(device)


@pytest.mark.parametrize("context,nodes,heads,kv", [(20000, 2, 1, 1), (17003, 64, 4, 2), (18001, 17, 2, 1)])
def test_contexts_joined_in_several_levels(device, context, nodes, heads, kv):
    """More than 64 stretches of an item, joined eight by eight by eight; pages that
    are not there in the midst of it, all positions of which are left out, and
    counted by halves of a tile: four to a page."""
    t = Trees([context], [nodes], heads, kv, 16, 64, torch.float16, 30)
    want = t.check(device)
    assert torch.equal(t.run(device), want)
    t.table[0, 100], t.table[0, 171] = -1, t.pages
    errors = torch.zeros(1, dtype=torch.int32, device=device)
    got = t.run(device, errors=errors)
    exact, err = t.exact()
    _within(got, exact, err, t.dt)
    assert int(errors) == 8


def test_many_heads_of_one_key_head(device):
    """64 heads of a key head and 64 nodes: 4096 rows."""
    Trees([40, 3], [64, 5], 64, 1, 64, 16, torch.bfloat16, 31).check(device)


def test_many_sequences_of_unequal_length(device):
    """130 sequences, more than twice the lanes of a wave, cut into stretches that
    cross them, one of them long."""
    contexts, counts = [(i * 29) % 70 for i in range(130)], [(i * 5) % 4 for i in range(130)]
    contexts[77], counts[77] = 5000, 3
    Trees(contexts, counts, 2, 1, 32, 16, torch.bfloat16, 32).check(device)


@pytest.mark.parametrize("long", [0, 4000])
@pytest.mark.parametrize("batch,heads,kv,hd", [(70, 6, 1, 64), (9, 8, 2, 128), (66, 12, 4, 32)])
def test_row_blocks_of_ragged_trees(device, batch, heads, kv, hd, long):
    """Trees of no, one and several row blocks side by side, more than 64 of them, with
    a long context among them (stretches) and without one (whole items)."""
    contexts, counts = [(i * 31) % 75 for i in range(batch)], [(i * 23) % 65 for i in range(batch)]
    contexts[batch // 2] += long
    counts[batch // 2] = 64
    Trees(contexts, counts, heads, kv, hd, 16, torch.bfloat16, 33).check(device)


@pytest.mark.parametrize("heads,kv,hd,most", [(8, 8, 64, 3), (16, 8, 128, 9), (32, 8, 64, 12), (32, 8, 128, 15), (9, 9, 48, 1)])
def test_more_items_than_workgroups(device, heads, kv, hd, most):
    """A wave has a sequence's key head for itself."""
    batch = 90
    contexts, counts = [(i * 41) % 420 for i in range(batch)], [1 + (i * 3) % most if i % 7 else 0 for i in range(batch)]
    contexts[5], counts[5] = 0, most
    t = Trees(contexts, counts, heads, kv, hd, 16, torch.bfloat16, 34)
    want = t.check(device)
    assert torch.equal(t.run(device), want)
    t.mask[t.cu[5]] = 0
    t.table[3, 2], t.table[8, 0] = -1, t.pages
    t.v[0], t.k[0] = float("nan"), float("inf")  # the page of nobody
    t.table = t.table[:, :13].contiguous()  # 208 positions
    errors = torch.zeros(1, dtype=torch.int32, device=device)
    got = t.run(device, errors=errors)
    exact, err = t.exact()
    _within(got, exact, err, t.dt)
    # halves of tiles of a lost page, which is one of 16, and each sequence that the table cuts off
    lost = sum(1 for b, col in ((3, 2), (8, 0)) if counts[b] and contexts[b] + counts[b] > 16 * col)
    assert int(errors) == lost + sum(1 for c, n in zip(contexts, counts) if n and c + n > 208)
    assert (got[int(t.cu[5])] == 0).all()


def test_many_sequences(device):
    """More sequences than lanes of a wave, ragged, some without nodes."""
    counts = [(i * 7) % 5 for i in range(150)]
    Trees([(i * 37) % 90 for i in range(150)], counts, 2, 1, 64, 16, torch.bfloat16, 2).check(device)


@pytest.mark.parametrize("spread", [8.0, 40.0])
def test_large_scores(device, spread):
    """Scores far apart: one key takes nearly all of a row."""
    Trees([700, 65], [5, 20], 4, 2, 64, 32, torch.bfloat16, 4, spread=spread).check(device)


def test_scale(device):
    Trees([120], [6], 4, 4, 64, 16, torch.float16, 6).check(device, scale=0.02)
    Trees([120], [6], 4, 4, 64, 16, torch.float16, 6).check(device, scale=-0.1)
    Trees([120], [6], 4, 4, 64, 16, torch.float16, 6).check(device, scale=0.0)


def test_rows_that_see_nothing(device):
    """No context and an empty mask: zeros; a node that does not see itself."""
    t = Trees([0, 0, 40], [4, 1, 3], 4, 2, 64, 16, torch.bfloat16, 8)
    t.mask[0], t.mask[1], t.mask[4], t.mask[6] = 0, 1, 0, 0
    got = t.check(device)
    assert (got[0] == 0).all() and (got[4] == 0).all() and (got[6] != 0).any()
    # bits past the tree's nodes are of no meaning
    want = t.run(device)
    t.mask |= torch.tensor([-1 << 10], dtype=torch.int64)
    assert torch.equal(t.run(device), want)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("heads,kv,hd", [(4, 4, 64), (8, 1, 128), (3, 1, 48)])
def test_what_is_not_seen_does_not_reach_a_row(device, bad, heads, kv, hd):
    """Keys and values behind the last node, in pages of nobody, and of nodes
    that some rows see and others do not."""
    t = Trees([50, 7], [9, 3], heads, kv, hd, 16, torch.bfloat16, 10)
    clean, err = t.exact()
    for b in range(2):
        end = t.contexts[b] + t.counts[b]
        page = t.table[b, (end - 1) // 16]
        t.k[page, :, (end - 1) % 16 + 1:] = bad
        t.v[page, :, (end - 1) % 16 + 1:] = bad
    t.k[0], t.v[0] = bad, bad
    t.check(device)
    # node 4 of the first tree: nobody but node 4 and its descendants see it
    x = 50 + 4
    page = t.table[0, x // 16]
    t.v[page, :, x % 16, ::3] = bad
    got = t.run(device)
    sees = [bool(int(t.mask[i]) >> 4 & 1) for i in range(9)] + [False] * 3
    assert any(sees) and not all(sees)
    rows = [i for i, s in enumerate(sees) if not s]
    _within(got[rows], clean[rows], err[rows], t.dt)
    seeing = got[[i for i, s in enumerate(sees) if s]].view(-1, heads, hd).float()
    assert not torch.isfinite(seeing[..., ::3]).any()
    keep = torch.ones(hd, dtype=torch.bool)
    keep[::3] = False
    assert torch.isfinite(seeing[..., keep.to(device)]).all()
    t.k[page, :, x % 16] = bad
    _within(t.run(device)[rows], clean[rows], err[rows], t.dt)


@pytest.mark.parametrize("entry", [-1, -2 ** 31, 2 ** 31 - 1, None])
def test_bad_pages(device, entry):
    """Positions whose page does not exist are left out and counted."""
    t = Trees([70, 40], [3, 20], 4, 2, 64, 16, torch.bfloat16, 12)
    entry = t.pages if entry is None else entry
    for b, col in ((0, 1), (0, 4), (1, 3)):
        t.table[b, col] = entry
    errors = torch.zeros(1, dtype=torch.int32, device=device)
    got = t.run(device, errors=errors)
    want, err = t.exact()
    _within(got, want, err, t.dt)
    assert int(errors) > 0
    assert torch.equal(t.run(device), got)


def test_short_block_table(device):
    """Contexts past the block table: what it covers counts."""
    t = Trees([40, 10], [4, 2], 2, 1, 64, 16, torch.bfloat16, 14)
    t.table = t.table[:, :2].contiguous()  # 32 positions
    errors = torch.zeros(1, dtype=torch.int32, device=device)
    want, err = t.exact()
    _within(t.run(device, errors=errors), want, err, t.dt)
    assert int(errors) > 0
    t.table = t.table[:, :0].contiguous()
    assert (t.run(device) == 0).all()


def test_rows_behind_the_last_sequence(device):
    """Rows that no sequence names stay as they are; counts past max_nodes or the
    rows, and offsets out of order, are cut off."""
    t = Trees([20, 30], [3, 4], 2, 2, 64, 16, torch.bfloat16, 16)
    want = t.run(device)
    t.q = torch.cat([t.q, t.q[:2]])
    t.mask = torch.cat([t.mask, t.mask[:2]])
    got = t.run(device, rows=12)
    assert torch.equal(got[:7], want) and (got[7:] == 7).all()
    cut = t.run(device, rows=9, max_nodes=2)
    assert (cut[[2, 5, 6, 7, 8]] == 7).all() and (cut[[0, 1, 3, 4]] != 7).any()
    t.cu = torch.tensor([0, 3, 100], dtype=torch.int32)
    wild = t.run(device, rows=9, max_nodes=64)
    assert torch.equal(wild[:3], want[:3]) and (wild[3:9] != 7).any(dim=1).all()
    t.cu = torch.tensor([5, 3, 7], dtype=torch.int32)
    assert (t.run(device, rows=9)[:3] == 7).all()
    t.ctx = torch.tensor([-5, -1], dtype=torch.int32)
    t.cu = torch.tensor([0, 3, 7], dtype=torch.int32)
    t.contexts = [0, 0]
    t.q, t.mask, t.t = t.q[:7], t.mask[:7], 7
    w, err = t.exact()
    _within(t.run(device), w, err, t.dt)


def test_attention_layouts(device):
    """Queries inside a packed row, a cache in [pages, page, heads, hd] order with
    padded rows, a wider output and table: the same bits."""
    t = Trees([90, 33], [5, 12], 4, 2, 64, 16, torch.float16, 18)
    want = t.run(device)
    packed = torch.full((t.t, 9, 64), float("nan"), dtype=t.dt, device=device)
    packed[:, 1:8:2] = t.q.to(device)
    caches = []
    for x in (t.k, t.v):
        whole = torch.full((t.pages, 16, 2, 72), float("nan"), dtype=t.dt, device=device)
        whole[..., :64] = x.to(device).transpose(1, 2)
        caches.append(whole[..., :64].transpose(1, 2))
    out = torch.full((t.t, 304), 7.0, dtype=t.dt, device=device)[:, 8:264]
    table = torch.full((2, 30), 2 ** 30, dtype=torch.int32, device=device)
    table[:, :t.table.shape[1]] = t.table.to(device)
    got = t.run(device, q=packed[:, 1:8:2], k_cache=caches[0], v_cache=caches[1], out=out,
                block_table=table[:, :t.table.shape[1]])
    assert torch.equal(got, want)


def test_attention_repeats(device):
    """The same bits again, with a workspace full of rubbish behind its counters,
    and on another stream than the tensors'; the counters are left at zero."""
    t = Trees([3000, 5, 777], [6, 1, 30], 8, 2, 128, 32, torch.bfloat16, 20)
    want = t.run(device)
    ws = ops.tree_attention_workspace(t.q.to(device), t.k, t.max_nodes)
    for fill in (0, 255):
        ws[12288:].fill_(fill)
        assert torch.equal(t.run(device, workspace=ws), want)
        assert (ws[:12288] == 0).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = t.run(device, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_far_offsets(device):
    """A cache of more than 2^32 bytes: pages at both of its ends."""
    kv, page, hd = 4, 64, 128
    pages = (9 << 30) // (kv * page * hd * 2) // 2 + 3
    k = torch.zeros(pages, kv, page, hd, dtype=torch.bfloat16, device=device)
    v = torch.zeros(pages, kv, page, hd, dtype=torch.bfloat16, device=device)
    t = Trees([130, 60], [3, 2], 8, kv, hd, page, torch.bfloat16, 22)
    want = t.run(device)
    far = torch.tensor([0] + list(range(pages - t.pages + 1, pages)))
    k[far.to(device)], v[far.to(device)] = t.k.to(device), t.v.to(device)
    table = torch.where(t.table < 0, t.table, far[t.table.clamp(min=0).long()].int())
    assert torch.equal(t.run(device, k_cache=k, v_cache=v, block_table=table.to(device)), want)
    # and the append to them
    slots = torch.tensor([pages * page - 1, (pages - 1) * page, 5], dtype=torch.int32, device=device)
    qkv = torch.randn(3, 8 + 2 * kv, hd, device=device, generator=None).to(torch.bfloat16)
    ops.rope_append(qkv, slots * 0, None, torch.empty(3, 8, hd, dtype=torch.bfloat16, device=device), k, v, slots)
    for i, (pg, r) in enumerate(((pages - 1, page - 1), (pages - 1, 0), (0, 5))):
        assert torch.equal(k[pg, :, r], qkv[i, 8:8 + kv]) and torch.equal(v[pg, :, r], qkv[i, 8 + kv:])


# ------------------------------------------------------------- verification

def _verify_oracle(p, q, tokens, parents, au, su, cu, n_max):
    """(path, count, token) by the definition, each residual normalised in its
    turn (None: no weight left)."""
    paths, counts, nexts = [], [], []
    weights = lambda row: row.double().nan_to_num(0).clamp(min=0)  # noqa: E731
    for b in range(len(cu) - 1):
        lo, n = cu[b], cu[b + 1] - cu[b]
        path, r = [0] if n else [], weights(p[lo]) if n else None
        for j in range(1, n):
            cur = path[-1]
            if parents[lo + j] != cur:
                continue
            x, d = tokens[lo + j], q[lo + cur].double()
            if r is not None and 0 <= x < p.shape[1] and float(au[lo + j].double() * d[x]) < float(r[x]):
                path.append(j)
                r = weights(p[lo + j])
            elif r is not None:
                r = weights(r - d)
                r = r / r.sum() if float(r.sum()) > 0 else None
        token = -1
        if n:
            r = weights(p[lo + path[-1]]) if r is None else r
            over = torch.nonzero(torch.cumsum(r, 0) > float(su[b].double()) * float(r.sum())).flatten()
            some = torch.nonzero(r > 0).flatten()
            token = int(over[0]) if over.numel() else int(some[-1]) if some.numel() else -1
        paths.append(path + [-1] * (n_max - len(path)))
        counts.append(len(path))
        nexts.append(token)
    return paths, counts, nexts


class Drafts:
    def __init__(self, counts, vocab, shape, seed, noise=0.7):
        g = _gen(seed)
        self.counts, t = counts, sum(counts)
        self.cu = [sum(counts[:b]) for b in range(len(counts) + 1)]
        logits = 3 * torch.randn(t, vocab, generator=g)
        self.p = torch.softmax(logits, 1)
        self.q = torch.softmax(logits + noise * torch.randn(t, vocab, generator=g), 1)
        self.parents = []
        for n in counts:
            self.parents += [-1] + [j - 1 if shape == "chain" else int(torch.randint((j - 1) // 4, (j + 1) // 2, (1,), generator=g))
                                    for j in range(1, n)] if n else []
        self.tokens = []
        for b, n in enumerate(counts):
            for j in range(n):
                row = self.q[self.cu[b] + max(self.parents[self.cu[b] + j], 0)]
                self.tokens.append(int(torch.multinomial(row, 1, generator=g)))
        self.au, self.su = torch.rand(t, generator=g), torch.rand(len(counts), generator=g)
        self.n_max = max(counts + [1])

    def run(self, device, rows=None, errors=None, p=None, q=None):
        b = len(self.counts)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
        path = torch.full((b, self.n_max + 3), 99, dtype=torch.int32, device=device)
        count, token = i32([99] * b), i32([99] * b)
        got = ops.verify_tree(self.p.to(device) if p is None else p, self.q.to(device) if q is None else q, i32(self.tokens),
                              i32(self.parents), self.au.to(device), self.su.to(device), path[:, :self.n_max], count, token,
                              cu_nodes=i32(self.cu), index_errors=errors)
        assert got is token and (path[:, self.n_max:] == 99).all()
        return path[:, :self.n_max].tolist(), count.tolist(), token.tolist()

    def want(self):
        return _verify_oracle(self.p, self.q, self.tokens, self.parents, self.au, self.su, self.cu, self.n_max)


@pytest.mark.parametrize("counts,vocab", [([1], 1), ([1, 2], 2), ([6, 6, 6, 6], 1000), ([9, 1, 0, 64, 17], 4099),
                                          ([5, 7], 70001), ([3] * 40, 257), ([12, 20, 3], 1024)])
@pytest.mark.parametrize("shape", ["chain", "tree"])
def test_verify(device, counts, vocab, shape):
    for seed in range(4):
        d = Drafts(counts, vocab, shape, seed, noise=(0.3, 0.7, 1.5, 4.0)[seed])
        assert d.run(device) == d.want()


def test_verify_keeps_the_distribution(device):
    """Two children of a root and a chain behind the first, 60000 times: the
    first token kept is distributed as the target's."""
    trials, vocab = 60000, 5
    g = _gen(1)
    p, q = torch.softmax(torch.randn(4, vocab, generator=g), 1), torch.softmax(torch.randn(4, vocab, generator=g), 1)
    tokens = torch.zeros(trials, 4, dtype=torch.int32)
    tokens[:, 1:3] = torch.multinomial(q[0], 2 * trials, replacement=True, generator=g).view(trials, 2).int()
    tokens[:, 3] = torch.multinomial(q[1], trials, replacement=True, generator=g).int()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    path = torch.empty(trials, 4, dtype=torch.int32, device=device)
    count, token = torch.empty_like(path[:, 0]).contiguous(), torch.empty_like(path[:, 0]).contiguous()
    ops.verify_tree(p.repeat(trials, 1).to(device), q.repeat(trials, 1).to(device), tokens.view(-1).to(device),
                    i32([-1, 0, 0, 1]).repeat(trials), torch.rand(4 * trials, generator=g).to(device),
                    torch.rand(trials, generator=g).to(device), path, count, token,
                    cu_nodes=i32(range(0, 4 * trials + 1, 4)))
    path, count, token = path.cpu().long(), count.cpu(), token.cpu()
    first = torch.where(count > 1, tokens.long().gather(1, path[:, 1:2].clamp(min=0)).flatten(), token.long())
    share = torch.bincount(first, minlength=vocab) / trials
    # five standard deviations of a share
    assert ((share - p[0]).abs() <= 5 * (p[0] * (1 - p[0]) / trials).sqrt()).all()


def test_verify_edges(device):
    """The numbers' ends, distributions that agree, one-hot ones, weights that
    are none, a token outside the vocabulary, the same token twice."""
    d = Drafts([5, 5, 5, 5, 5, 5, 5, 5], 300, "tree", 3)
    d.au[:5], d.su[0] = 0.0, 0.0
    d.au[5:10], d.su[1] = 1 - 2.0 ** -24, 1 - 2.0 ** -24
    d.q[10:15] = d.p[10:15]
    d.p[15:20] = 0
    d.p[15:20, 17] = 1
    d.p[20:25, ::2] = float("nan")
    d.p[25:30] = 0
    d.tokens[31], d.tokens[32] = -1, 300
    d.tokens[36] = d.tokens[37] = d.tokens[38]
    errors = torch.zeros(1, dtype=torch.int32, device=device)
    got = d.run(device, errors=errors)
    assert got == d.want()
    assert got[2][3] == 17 and got[2][5] == -1 and int(errors) > 0
    # no residual left: p below q everywhere, every child refused, so p itself
    e = Drafts([3], 64, "chain", 5)
    e.q[0], e.p[0] = 1 / 64, 1 / 128
    e.au[:] = 0.9
    assert e.run(device) == e.want() and e.run(device)[1] == [1]


@pytest.mark.parametrize("counts,vocab", [([20, 9], 128257), ([30], 300001), ([5] * 100, 33000)])
def test_verify_over_several_workgroups(device, counts, vocab):
    for seed in range(2):
        d = Drafts(counts, vocab, "tree", seed, noise=(1.0, 4.0)[seed])
        assert d.run(device) == d.want()


def test_verify_strides_and_bad_offsets(device):
    d = Drafts([6, 9, 4], 500, "tree", 7)
    want = d.run(device)
    wide_p = torch.full((19, 640), 9.0, device=device)
    wide_q = torch.full((19, 700), 9.0, device=device)
    wide_p[:, 3:503], wide_q[:, 100:600] = d.p.to(device), d.q.to(device)
    assert d.run(device, p=wide_p[:, 3:503], q=wide_q[:, 100:600]) == want
    d.cu = [0, 6, 15, 1000]
    assert d.run(device) == want  # cut off at the rows
    d.cu = [-3, 6, 15, 19]
    assert d.run(device)[1][1:] == want[1][1:]
    d.cu, (a, b, c) = [0, 6, 6, 2], want
    path, count, token = d.run(device)
    assert path[0] == a[0] and count == [b[0], 0, 0] and token == [c[0], -1, -1]
    assert path[1] == path[2] == [-1] * 9
    # parents that are none of a tree's: nodes that are never reached
    d = Drafts([5], 50, "chain", 9, noise=0.0)
    d.parents = [0, 1, 7, -5, 3]
    assert d.run(device) == d.want() and d.run(device)[1] == [1]


def test_verify_offsets_at_the_ends_of_32_bits(device):
    """An offset of -2^31 behind a positive one: no nodes."""
    d = Drafts([6, 9, 4], 500, "tree", 7)
    path, count, token = d.run(device)
    d.cu = [0, 6, -2 ** 31, 2 ** 31 - 1]
    got = d.run(device)
    assert got[0][0] == path[0] and got[0][1] == [-1] * 9
    assert got[1][:2] == [count[0], 0] and got[2][:2] == [token[0], -1]


# --------------------------------------------------------------- compaction

@pytest.mark.parametrize("layers,kv,hd,page", [(1, 1, 16, 16), (3, 4, 64, 16), (2, 2, 128, 32), (1, 3, 80, 16), (5, 2, 48, 64)])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_compact(device, layers, kv, hd, page, dt):
    contexts, counts = [0, 13, 16, 100, 31, 5], [64, 40, 3, 12, 64, 1]
    t = Trees(contexts, counts, kv, kv, hd, page, DT[dt], layers)
    g = _gen(hd)
    k = torch.randn(layers, *t.k.shape, generator=g).to(DT[dt])
    v = torch.randn(layers, *t.k.shape, generator=g).to(DT[dt])
    path = torch.full((6, 64), -1, dtype=torch.int32)
    count = torch.tensor([64, 9, 2, 5, 40, 1], dtype=torch.int32)
    for b, n in enumerate(counts):
        m = int(count[b])
        path[b, 0] = 0
        path[b, 1:m] = (1 + torch.randperm(n - 1, generator=g)[:m - 1]).sort().values.int() if n > 1 else 0
    want_k, want_v = k.clone(), v.clone()
    at = lambda b, x: (t.table[b, x // page].long(), x % page)  # noqa: E731
    for b in range(6):
        for i in range(1, int(count[b])):
            (sp, sr), (dp, dr) = at(b, contexts[b] + int(path[b, i])), at(b, contexts[b] + i)
            want_k[:, dp, :, dr], want_v[:, dp, :, dr] = k[:, sp, :, sr], v[:, sp, :, sr]
    dk, dv = k.to(device), v.to(device)
    errors = torch.zeros(1, dtype=torch.int32, device=device)
    args = [x.to(device) for x in (t.table, t.ctx, path, count)]
    if layers == 1:
        ops.compact_cache(dk[0], dv[0], *args, index_errors=errors)
    else:
        ops.compact_cache(dk, dv, *args, index_errors=errors)
    assert torch.equal(dk.cpu(), want_k) and torch.equal(dv.cpu(), want_v) and int(errors) == 0


def test_compact_bad_entries(device):
    """Entries that no tree can have and pages that do not exist move nothing and
    are counted; counts past the path are cut off."""
    t = Trees([20, 30, 10], [8, 8, 8], 2, 2, 64, 16, torch.bfloat16, 3)
    path = torch.tensor([[0, 2, 1, 64, 7, -1, 6, 7], [0, 3, 4, 5, 6, 7, 7, 7], [0, 1, 2, 3, 4, 5, 6, 7]], dtype=torch.int32)
    count = torch.tensor([6, -3, 100], dtype=torch.int32)
    k, v = t.k.to(device), t.v.to(device)
    errors = torch.zeros(1, dtype=torch.int32, device=device)
    ops.compact_cache(k, v, t.table.to(device), t.ctx.to(device), path.to(device), count.to(device), index_errors=errors)
    want_k, want_v = t.k.clone(), t.v.clone()
    for i in (1, 4):  # 2 -> 1 and 7 -> 4; 1 < 2, 64 and -1 are refused
        (sp, sr), (dp, dr) = divmod(20 + int(path[0, i]), 16), divmod(20 + i, 16)
        for w, x in ((want_k, t.k), (want_v, t.v)):
            w[t.table[0, dp].long(), :, dr] = x[t.table[0, sp].long(), :, sr]
    assert torch.equal(k.cpu(), want_k) and torch.equal(v.cpu(), want_v) and int(errors) == 3
    table = t.table.clone()
    table[0, 1] = t.pages
    ops.compact_cache(k, v, table.to(device)[:, :2], t.ctx.to(device), path.to(device), count.to(device), index_errors=errors)
    # none of the first tree's five: three of before, two by their page
    assert torch.equal(k.cpu(), want_k)
    assert int(errors) == 3 + 5
