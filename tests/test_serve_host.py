"""What the serving operators refuse, through the C-ABI and the Python wrappers
(no GPU: every call is rejected before a launch), and the rotation's table."""

import ctypes

import pytest
import torch

from tjkernels import _lib, ops
from tjkernels._lib import BF16, EINVAL, EUNSUPPORTED, F16, F32, PagedCache, TjkError

FAKE = 1 << 20  # a pointer that is never followed


def _cache(**kw):
    a = dict(k=FAKE, v=FAKE, page_stride=4 * 32 * 64, head_stride=32 * 64, row_stride=64, pages=10, page_size=32, kv_heads=4,
             head_dim=64, dtype=BF16)
    a.update(kw)
    return PagedCache(*a.values())


def _call(name, a, kw):
    cache = {k[6:]: v for k, v in kw.items() if k.startswith("cache_")}
    a.update({k: v for k, v in kw.items() if not k.startswith("cache_")})
    if "cache" in a and a["cache"] is not None:
        a["cache"] = ctypes.byref(_cache(**cache))
    return getattr(_lib.load(), name)(*a.values())


def _append(**kw):
    return _call("tjk_rope_append", dict(
        qkv=FAKE, ld_token=1024, ld_head=64, positions=FAKE, table=FAKE, n_positions=100, rot=64, interleaved=0,
        q_out=FAKE + 4096, ld_q_token=512, ld_q_head=64, k_out=None, ld_k_token=0, ld_k_head=0, cache=1, slots=FAKE,
        q_gamma=FAKE, k_gamma=None, eps=1e-6, index_errors=None, tokens=5, heads=8, kv_heads=4, head_dim=64, dtype=BF16,
        stream=None), kw)


def _attend(**kw):
    return _call("tjk_tree_attention", dict(
        q=FAKE, ld_q_token=512, ld_q_head=64, cache=1, table=FAKE, ld_table=8, table_cols=8, ctx_lens=FAKE, cu_nodes=FAKE,
        tree_mask=FAKE, out=FAKE, ld_out=512, tokens=5, batch=2, heads=8, max_nodes=4, scale=0.1, workspace=FAKE,
        workspace_bytes=1 << 40, index_errors=None, stream=None), kw)


def _verify(**kw):
    return _call("tjk_verify_tree", dict(
        target=FAKE, ld_target=100, draft=FAKE, ld_draft=100, tokens=FAKE, parents=FAKE, accept_u=FAKE, sample_u=FAKE,
        cu_nodes=FAKE, path=FAKE, ld_path=4, count=FAKE, token=FAKE, index_errors=None, rows=5, vocab=100, batch=2,
        max_nodes=4, workspace=FAKE, workspace_bytes=1 << 40, stream=None), kw)


def _compact(**kw):
    return _call("tjk_compact_cache", dict(
        cache=1, layers=2, layer_stride=1 << 20, table=FAKE, ld_table=8, table_cols=8, ctx_lens=FAKE, path=FAKE, ld_path=4,
        max_nodes=4, count=FAKE, index_errors=None, batch=2, stream=None), kw)


def _said():
    return _lib.load().tjk_last_error_string().decode()


BAD_CACHES = [
    (dict(cache_k=None), EINVAL, "null"), (dict(cache_v=None), EINVAL, "null"), (dict(cache_dtype=F32), EINVAL, "dtype"),
    (dict(cache_kv_heads=0), EINVAL, "shape"), (dict(cache_pages=-1), EINVAL, "shape"),
    (dict(cache_head_dim=72), EUNSUPPORTED, "multiple of 16"), (dict(cache_head_dim=144), EUNSUPPORTED, "128"),
    (dict(cache_page_size=8), EUNSUPPORTED, "power of two"), (dict(cache_page_size=48), EUNSUPPORTED, "power of two"),
    (dict(cache_page_size=1 << 17), EUNSUPPORTED, "power of two"),
    (dict(cache_pages=1 << 26, cache_page_size=32), EUNSUPPORTED, "int32"), (dict(cache_row_stride=56), EINVAL, "strides"),
    (dict(cache_page_stride=-64), EINVAL, "strides"), (dict(cache_head_stride=100), EUNSUPPORTED, "multiples of 8"),
    (dict(cache_row_stride=1 << 21), EUNSUPPORTED, "too large"), (dict(cache_k=FAKE + 8), EUNSUPPORTED, "misaligned"),
]


@pytest.mark.parametrize("call", [_append, _attend, _compact])
@pytest.mark.parametrize("kw,status,word", BAD_CACHES)
def test_cache_refusals(call, kw, status, word):
    assert call(**kw) == status and word in _said()


@pytest.mark.parametrize("kw,status,word", [
    (dict(tokens=-1), EINVAL, "shape"), (dict(heads=0), EINVAL, "shape"), (dict(kv_heads=0), EINVAL, "shape"),
    (dict(dtype=F32), EINVAL, "dtype"), (dict(dtype=F16), EINVAL, "differ"), (dict(kv_heads=2), EINVAL, "differ"),
    (dict(head_dim=40), EUNSUPPORTED, "multiple of 16"), (dict(rot=24), EUNSUPPORTED, "rotated"),
    (dict(rot=80), EUNSUPPORTED, "rotated"), (dict(tokens=1 << 31), EUNSUPPORTED, "large"),
    (dict(qkv=None), EINVAL, "null"), (dict(positions=None), EINVAL, "null"), (dict(table=None), EINVAL, "null"),
    (dict(q_out=None), EINVAL, "null"), (dict(slots=None), EINVAL, "null"), (dict(cache=None), EINVAL, "null"),
    (dict(ld_head=56), EINVAL, "stride"), (dict(ld_q_head=0), EINVAL, "stride"), (dict(ld_token=1020), EUNSUPPORTED, "8"),
    (dict(ld_q_token=516), EUNSUPPORTED, "8"), (dict(k_out=FAKE + 64, ld_k_head=64, ld_k_token=4), EUNSUPPORTED, "8"),
    (dict(qkv=FAKE + 8), EUNSUPPORTED, "misaligned"), (dict(table=FAKE + 4), EUNSUPPORTED, "misaligned"),
    (dict(q_out=FAKE), EINVAL, "in place"), (dict(k_out=FAKE, ld_k_head=64, ld_k_token=1024), EINVAL, "in place"),
    (dict(k_out=FAKE + 2 * 8 * 64, ld_k_head=64, ld_k_token=256), EINVAL, "in place"),
])
def test_append_refusals(kw, status, word):
    assert _append(**kw) == status and word in _said()


@pytest.mark.parametrize("kw,status,word", [
    (dict(tokens=-1), EINVAL, "shape"), (dict(batch=-1), EINVAL, "shape"), (dict(heads=0), EINVAL, "shape"),
    (dict(max_nodes=-1), EINVAL, "shape"), (dict(heads=6), EINVAL, "multiple"), (dict(max_nodes=65), EUNSUPPORTED, "64"),
    (dict(tokens=1 << 31), EUNSUPPORTED, "large"), (dict(batch=1 << 24), EUNSUPPORTED, "large"),
    (dict(q=None), EINVAL, "null"), (dict(out=None), EINVAL, "null"), (dict(ctx_lens=None), EINVAL, "null"),
    (dict(cu_nodes=None), EINVAL, "null"), (dict(table=None), EINVAL, "null"), (dict(ld_table=7), EINVAL, "leading"),
    (dict(ld_out=504), EINVAL, "leading"), (dict(ld_q_head=56), EINVAL, "leading"),
    (dict(ld_q_token=513), EUNSUPPORTED, "multiples of 8"), (dict(ld_out=516), EUNSUPPORTED, "multiples of 8"),
    (dict(q=FAKE + 8), EUNSUPPORTED, "misaligned"), (dict(tree_mask=FAKE + 4), EUNSUPPORTED, "misaligned"),
    (dict(workspace=FAKE + 8), EUNSUPPORTED, "misaligned"),
])
def test_attention_refusals(kw, status, word):
    assert _attend(**kw) == status and word in _said()


def test_attention_refuses_a_small_workspace():
    need = _lib.load().tjk_tree_attention_bytes(8, 4, 64, 4)
    if need:
        assert _attend(workspace_bytes=need - 1) == EINVAL and "workspace" in _said()
        assert _attend(workspace=None) == EINVAL and "null" in _said()
    for bad in ((0, 1, 64, 4), (8, 0, 64, 4), (8, 3, 64, 4), (8, 4, 72, 4), (8, 4, 64, 65), (8, 4, 64, 0)):
        assert _lib.load().tjk_tree_attention_bytes(*bad) == 0


@pytest.mark.parametrize("kw,status,word", [
    (dict(rows=-1), EINVAL, "shape"), (dict(vocab=0), EINVAL, "shape"), (dict(batch=-1), EINVAL, "shape"),
    (dict(max_nodes=0), EINVAL, "shape"), (dict(max_nodes=65, ld_path=65), EUNSUPPORTED, "64"),
    (dict(vocab=1 << 25, ld_target=1 << 25, ld_draft=1 << 25), EUNSUPPORTED, "large"),
    (dict(rows=1 << 31), EUNSUPPORTED, "large"), (dict(target=None), EINVAL, "null"), (dict(path=None), EINVAL, "null"),
    (dict(sample_u=None), EINVAL, "null"), (dict(parents=None), EINVAL, "null"), (dict(ld_draft=99), EINVAL, "leading"),
    (dict(ld_path=3), EINVAL, "leading"), (dict(workspace=FAKE + 8), EUNSUPPORTED, "misaligned"),
])
def test_verify_refusals(kw, status, word):
    assert _verify(**kw) == status and word in _said()


def test_verify_refuses_a_small_workspace():
    big = dict(vocab=200000, ld_target=200000, ld_draft=200000)
    need = _lib.load().tjk_verify_tree_bytes(200000, 2)
    assert need > 0 and _lib.load().tjk_verify_tree_bytes(100, 2) == 0
    assert _verify(workspace_bytes=need - 1, **big) == EINVAL and "workspace" in _said()
    assert _verify(workspace=None, **big) == EINVAL and "workspace" in _said()
    for bad in ((0, 2), (100000, 0), (1 << 25, 2)):
        assert _lib.load().tjk_verify_tree_bytes(*bad) == 0


@pytest.mark.parametrize("kw,status,word", [
    (dict(layers=-1), EINVAL, "shape"), (dict(batch=-1), EINVAL, "shape"), (dict(max_nodes=65), EUNSUPPORTED, "64"),
    (dict(layer_stride=4), EUNSUPPORTED, "8"), (dict(table=None), EINVAL, "null"), (dict(path=None), EINVAL, "null"),
    (dict(count=None), EINVAL, "null"), (dict(ld_table=7), EINVAL, "leading"), (dict(ld_path=3), EINVAL, "leading"),
])
def test_compact_refusals(kw, status, word):
    assert _compact(**kw) == status and word in _said()


def test_nothing_to_do_is_no_error():
    assert _append(tokens=0, qkv=None) == 0
    assert _attend(tokens=0, q=None) == 0 and _attend(batch=0, q=None) == 0 and _attend(max_nodes=0, q=None) == 0
    assert _verify(batch=0, path=None) == 0
    assert _compact(batch=0, path=None) == 0 and _compact(layers=0) == 0 and _compact(max_nodes=1) == 0


# ------------------------------------------------------------ Python wrappers

def _b(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def _i(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def _py_append(**kw):
    a = dict(qkv=_b(5, 16, 64), positions=_i(5), table=torch.zeros(100, 32, 2), q_out=_b(5, 8, 64), k_cache=_b(10, 4, 32, 64),
             v_cache=_b(10, 4, 32, 64), slots=_i(5), k_out=_b(5, 4, 64), q_gamma=torch.ones(64), k_gamma=torch.ones(64))
    a.update(kw)
    ops.rope_append(**a)


def _py_attend(**kw):
    a = dict(q=_b(5, 8, 64), k_cache=_b(10, 4, 32, 64), v_cache=_b(10, 4, 32, 64), block_table=_i(2, 8), ctx_lens=_i(2),
             out=_b(5, 512), cu_nodes=_i(3), max_nodes=4, tree_mask=torch.zeros(5, dtype=torch.int64))
    a.update(kw)
    ops.tree_attention(**a)


def _py_verify(**kw):
    a = dict(target=torch.zeros(5, 100), draft=torch.zeros(5, 100), tokens=_i(5), parents=_i(5), accept_u=torch.zeros(5),
             sample_u=torch.zeros(2), path=_i(2, 4), count=_i(2), token=_i(2), cu_nodes=_i(3))
    a.update(kw)
    ops.verify_tree(**a)


def _py_compact(**kw):
    a = dict(k_cache=_b(3, 10, 4, 32, 64), v_cache=_b(3, 10, 4, 32, 64), block_table=_i(2, 8), ctx_lens=_i(2), path=_i(2, 4),
             count=_i(2))
    a.update(kw)
    ops.compact_cache(**a)


@pytest.mark.parametrize("call", [_py_append, _py_attend, _py_verify, _py_compact])
def test_wrappers_take_device_tensors_only(call):
    with pytest.raises(TjkError, match="device tensors"):
        call()


def test_well_formed_layouts():
    """Permuted caches, padded rows, single heads, tokens and pages of any
    stride, no cache, no table, in place: refused last, for the device."""
    wide = _b(10, 32, 4, 72)
    packed = _b(5, 3, 4, 64)
    flat = packed.view(5, 12, 64)
    for kw in (dict(k_cache=wide[..., :64].transpose(1, 2), v_cache=wide[..., :64].transpose(1, 2)),
               dict(k_cache=_b(1, 4, 32, 64), v_cache=_b(3, 4, 32, 64)[::3]), dict(k_out=None), dict(table=None),
               dict(k_cache=None, v_cache=None, slots=None), dict(q_gamma=None), dict(q_out=_b(9, 8, 80)[:7, :, :64]),
               dict(qkv=flat, q_out=flat[:, :4], k_out=flat[:, 4:8]),
               dict(qkv=_b(5, 3, 64), q_out=_b(5, 1, 64), k_out=_b(5, 1, 64), k_cache=_b(10, 1, 32, 64),
                    v_cache=_b(10, 1, 32, 64))):
        with pytest.raises(TjkError, match="device tensors"):
            _py_append(**kw)
    for kw in (dict(tree_mask=None), dict(q=_b(5, 16, 64)[:, ::2]), dict(out=_b(9, 600)[2:, :512]),
               dict(block_table=_i(2, 16)[:, :3]), dict(workspace=torch.zeros(1 << 27, dtype=torch.uint8))):
        with pytest.raises(TjkError, match="device tensors"):
            _py_attend(**kw)
    for kw in (dict(target=torch.zeros(5, 128)[:, :100]), dict(path=_i(2, 9)[:, :4])):
        with pytest.raises(TjkError, match="device tensors"):
            _py_verify(**kw)
    for kw in (dict(k_cache=_b(10, 4, 32, 64), v_cache=_b(10, 4, 32, 64)), dict(path=_i(2, 9)[:, :4])):
        with pytest.raises(TjkError, match="device tensors"):
            _py_compact(**kw)


@pytest.mark.parametrize("kw,word", [
    (dict(qkv=_b(5, 1024)), "qkv must be"), (dict(qkv=_b(5, 64, 16).transpose(1, 2)), "qkv must be"),
    (dict(qkv=torch.zeros(5, 16, 64, dtype=torch.float64)), "dtype"), (dict(q_out=_b(5, 16, 64)), "left"),
    (dict(q_out=_b(5, 7, 64)), "left"), (dict(q_out=_b(4, 8, 64)), "q_out must be"), (dict(q_out=_b(5, 8, 32)), "q_out"),
    (dict(q_out=torch.zeros(5, 8, 64, dtype=torch.float16)), "q_out"), (dict(k_out=_b(5, 3, 64)), "k_out"),
    (dict(positions=_i(4)), "positions"), (dict(positions=torch.zeros(5, dtype=torch.int64)), "positions"),
    (dict(table=torch.zeros(100, 64)), "table"), (dict(table=torch.zeros(100, 2, 32).transpose(1, 2)), "table"),
    (dict(table=_b(100, 32, 2)), "table"), (dict(slots=None), "together"), (dict(v_cache=None), "together"),
    (dict(slots=_i(6)), "slots"), (dict(k_cache=_b(10, 4, 16, 64)), "differ"),
    (dict(k_cache=_b(10, 32, 4, 64).transpose(1, 2)), "strides"), (dict(k_cache=_b(1, 10, 4, 32, 64)), "k_cache must be"),
    (dict(q_gamma=torch.ones(32)), "q_gamma"), (dict(k_gamma=_b(64)), "k_gamma"),
    (dict(index_errors=torch.zeros(1)), "index_errors"), (dict(qkv=None), "must be a tensor"),
])
def test_append_wrapper_refusals(kw, word):
    with pytest.raises(TjkError, match=word):
        _py_append(**kw)


@pytest.mark.parametrize("kw,word", [
    (dict(q=_b(5, 8, 32)), "differ"), (dict(q=torch.zeros(5, 8, 64, dtype=torch.float16)), "differ"),
    (dict(out=_b(5, 256)), "out must be"), (dict(out=_b(4, 512)), "out must be"), (dict(out=torch.zeros(5, 512)), "out must be"),
    (dict(block_table=_i(2, 8).long()), "block_table"), (dict(block_table=_i(8, 2).t()), "block_table"),
    (dict(ctx_lens=_i(3)), "ctx_lens"), (dict(cu_nodes=_i(2)), "cu_nodes"), (dict(tree_mask=_i(5)), "tree_mask"),
    (dict(tree_mask=torch.zeros(6, dtype=torch.int64)), "tree_mask"), (dict(max_nodes=1 << 33, workspace=_i(4)), "max_nodes"),
    (dict(workspace=torch.zeros(4, 4).t()), "workspace"), (dict(index_errors=_i(0)), "index_errors"),
])
def test_attention_wrapper_refusals(kw, word):
    with pytest.raises(TjkError, match=word):
        _py_attend(**kw)


@pytest.mark.parametrize("kw,word", [
    (dict(target=_b(5, 100)), "target"), (dict(draft=torch.zeros(5, 99)), "differ"), (dict(draft=torch.zeros(4, 100)), "differ"),
    (dict(target=torch.zeros(100, 5).t()), "target"), (dict(tokens=_i(4)), "tokens"), (dict(parents=_i(5).long()), "parents"),
    (dict(accept_u=torch.zeros(5, dtype=torch.float64)), "accept_u"), (dict(sample_u=torch.zeros(3)), "sample_u"),
    (dict(path=_i(4, 2).t()), "path"), (dict(count=_i(3)), "count"), (dict(token=_i(2).long()), "token"),
    (dict(cu_nodes=_i(4)), "cu_nodes"),
])
def test_verify_wrapper_refusals(kw, word):
    with pytest.raises(TjkError, match=word):
        _py_verify(**kw)


@pytest.mark.parametrize("kw,word", [
    (dict(k_cache=_b(3, 10, 4, 32, 64)[:2]), "differ"), (dict(k_cache=_b(1, 3, 10, 4, 32, 64)), "k_cache must be"),
    (dict(path=_i(3, 4)), "path"), (dict(count=_i(3)), "count"), (dict(ctx_lens=_i(1)), "ctx_lens"),
])
def test_compact_wrapper_refusals(kw, word):
    with pytest.raises(TjkError, match=word):
        _py_compact(**kw)


def test_rope_table():
    t = ops.rope_table(100000, 64, 500.0)
    assert t.shape == (100000, 32, 2) and t.dtype == torch.float32 and t.is_contiguous()
    x = torch.tensor([0, 1, 77, 99999], dtype=torch.float64)
    for i in (0, 5, 31):
        angle = x * 500.0 ** (-2 * i / 64)
        got = t[x.long(), i].double()
        # a step of the table, and the error of the 64-bit angle itself
        assert (got[:, 0] - angle.cos()).abs().max() <= 2.0 ** -25 + 1e-10
        assert (got[:, 1] - angle.sin()).abs().max() <= 2.0 ** -25 + 1e-10
    assert ops.rope_table(7, 0).shape == (7, 0, 2)
    with pytest.raises(TjkError, match="pairs"):
        ops.rope_table(8, 7)


def test_append_in_place_of_one_head():
    """In place, the head stride of a single head is of no meaning: with that in order
    the call is found too large, the last thing looked at."""
    one = dict(q_out=FAKE, cache=None, slots=None, heads=1, kv_heads=16, tokens=1 << 30, head_dim=128, rot=0, ld_head=136,
               ld_token=4488, ld_q_token=4488, ld_q_head=128)
    assert _append(**one) == EUNSUPPORTED and "too many" in _said()
    assert _append(**dict(one, ld_q_token=4480)) == EINVAL and "in place" in _said()


def test_attention_refuses_more_work_than_32_bits_number():
    """63 items of 34087042 units are 2^31 - 2, which the division among the
    workgroups, rounding up, would carry past 32 bits."""
    kw = dict(batch=63, heads=1, cache_kv_heads=1, ld_table=1 << 26)
    assert _attend(table_cols=34087042 - 8, **kw) == EUNSUPPORTED and "too large" in _said()


@pytest.mark.parametrize("call", [_append, _compact])
@pytest.mark.parametrize("kw", [dict(cache_page_stride=0), dict(cache_head_stride=0), dict(cache_head_stride=32)])
def test_written_caches_do_not_overlap(call, kw):
    assert call(**kw) == EINVAL and "overlap" in _said()
    assert _attend(workspace=None, **kw) == EINVAL and "null workspace" in _said()  # one that is read may


def test_outputs_do_not_overlap():
    assert _append(ld_q_token=0) == EINVAL and "stride" in _said()
    assert _append(k_out=FAKE + 64, ld_k_head=64, ld_k_token=0) == EINVAL and "stride" in _said()
    assert _compact(layer_stride=0) == EUNSUPPORTED and "row" in _said()
    assert _attend(q=FAKE, out=FAKE) == EINVAL and "out may not be q" in _said()


def test_wrappers_refuse_expanded_outputs():
    with pytest.raises(TjkError):
        _py_append(q_out=_b(1, 8, 64).expand(5, 8, 64))
    with pytest.raises(TjkError):
        _py_compact(k_cache=_b(1, 10, 4, 32, 64).expand(3, 10, 4, 32, 64), v_cache=_b(1, 10, 4, 32, 64).expand(3, 10, 4, 32, 64))


@pytest.mark.parametrize("kw", [dict(q=_b(5, 512)), dict(k_cache=_b(10, 32, 64)), dict(q=_b(5)), dict(q=_b(1, 5, 8, 64))])
def test_attention_shapes_are_refused_before_the_workspace(kw):
    with pytest.raises(TjkError):
        _py_attend(**kw)
    with pytest.raises(TjkError):
        _py_attend(workspace=torch.zeros(64, dtype=torch.uint8), **kw)


# ------------------------------------------------------------ rows that overlap

def _starts(base, *steps):
    at = [base]
    for stride, n in steps:
        at = [x + i * stride for x in at for i in range(n)]
    return at


def _overlap(rows, size):
    rows = sorted(rows)
    return any(b - a < size for a, b in zip(rows, rows[1:]))


# with every other check passed, the last thing looked at: too many tokens
MANY = dict(qkv=1 << 40, tokens=1 << 30, heads=1, kv_heads=16, head_dim=128, rot=0, ld_token=33 * 128, ld_head=128,
            q_out=1 << 50, ld_q_token=128, ld_q_head=128, cache=None, slots=None)


def test_written_caches_of_any_strides():
    """A cache is refused if two of its rows share an element, and only then."""
    g = torch.Generator()
    g.manual_seed(0)
    r = lambda n: int(torch.randint(0, n, (1,), generator=g))  # noqa: E731
    found = [0, 0]
    for _ in range(3000):
        hd, heads, pages = 16 * (1 + r(3)), 1 + r(4), 1 + r(5)
        short, wide = hd + 8 * r(4), hd + 8 * r(60)
        strides = [short, wide, (heads + r(2)) * short if r(2) else wide * 16 + 8 * r(3)]
        order = torch.randperm(3, generator=g).tolist()
        page, head, row = [strides[i] for i in order]
        bad = _overlap(_starts(0, (page, pages), (head, heads), (row, 16)), hd)
        kw = dict(cache=1, cache_k=1 << 53, cache_v=1 << 54, cache_page_stride=page, cache_head_stride=head, cache_row_stride=row,
                  cache_pages=pages, cache_page_size=16, cache_kv_heads=heads, cache_head_dim=hd)
        many = dict(MANY, slots=FAKE, head_dim=hd, kv_heads=heads, heads=1000, ld_head=hd, ld_token=(1000 + 2 * heads) * hd,
                    ld_q_token=1000 * hd, ld_q_head=hd, tokens=1 << 28, **kw)
        status = _append(**many)
        said = _said()
        assert (status == EINVAL and "rows of the cache overlap" in said) if bad else \
            (status == EUNSUPPORTED and "too many" in said), (page, head, row, pages, heads, hd, said)
        layer = 8 * (hd // 8 + r(pages * 16 * heads * 16))
        bad = _overlap(_starts(0, (layer, 3), (page, pages), (head, heads), (row, 16)), hd)
        status = _compact(layers=3, layer_stride=layer, batch=1 << 25, **kw)
        said = _said()
        assert (status == EINVAL and "rows of the cache overlap" in said) if bad else \
            (status == EUNSUPPORTED and "too large" in said), (layer, page, head, row, pages, heads, hd, said)
        found[bad] += 1
    assert min(found) > 100


def test_pages_whose_keys_are_values():
    cache = dict(cache=1, slots=FAKE, heads=1000, kv_heads=4, ld_token=1008 * 64, ld_head=64, head_dim=64, ld_q_token=64000,
                 ld_q_head=64, tokens=1 << 28, cache_k=1 << 53)
    many = {k: v for k, v in MANY.items() if k not in cache}
    rows = 2 * 64  # bytes
    for apart, bad in ((0, True), (rows - 16, True), (rows, True), (31 * rows, True), (128 * rows, False), (-rows, True),
                       (-128 * rows, False), (127 * rows + 16, True), (10 * 128 * rows, False)):
        status = _append(**many, **cache, cache_v=(1 << 53) + apart)
        assert (status == EINVAL and "keys and values overlap" in _said()) if bad else \
            (status == EUNSUPPORTED and "too many" in _said()), (apart, _said())


def test_outputs_beside_their_inputs():
    """q_out and k_out may lie in one buffer with qkv, between its rows, but in no
    place of theirs or of each other's other than their own."""
    g = torch.Generator()
    g.manual_seed(1)
    r = lambda n: int(torch.randint(0, n, (1,), generator=g))  # noqa: E731
    many = dict(MANY, head_dim=16, heads=700, kv_heads=50, tokens=1 << 28)
    found = [0, 0]
    for _ in range(1500):
        token = 16 * (800 + r(2) * 800)
        kw = dict(ld_token=token, ld_head=16, ld_q_token=token, ld_q_head=16, k_out=None, ld_k_token=token, ld_k_head=16)
        at = 8 * r(2 * token // 8)
        kw["q_out"] = MANY["qkv"] + 2 * (0 if r(8) == 0 else at)
        if r(2):
            kw["k_out"] = MANY["qkv"] + 2 * (700 * 16 if r(3) == 0 else 8 * r(2 * token // 8))
        # whether rows meet depends on the difference of their tokens: seven say all
        pieces = lambda p, n: {x // 8 + i for x in _starts((p - MANY["qkv"]) // 2, (token, 7), (16, n)) for i in (0, 1)}  # noqa: E731
        qkv, q = pieces(MANY["qkv"], 800), pieces(kw["q_out"], 700)
        k = pieces(kw["k_out"], 50) if kw["k_out"] else set()
        bad = (kw["q_out"] != MANY["qkv"] and q & qkv) or (kw["k_out"] != MANY["qkv"] + 2 * 700 * 16 and k & qkv) or q & k
        if kw["k_out"] == MANY["qkv"]:
            bad = True
        status = _append(**dict(many, **kw))
        assert (status == EINVAL) if bad else (status == EUNSUPPORTED and "too many" in _said()), (kw, _said())
        found[bool(bad)] += 1
    assert min(found) > 30


def test_outputs_whose_own_rows_overlap():
    for kw, bad in ((dict(heads=4, ld_q_token=256, ld_q_head=128), True), (dict(heads=4, ld_q_token=512, ld_q_head=128), False),
                    (dict(heads=4, ld_q_token=128, ld_q_head=128 << 30), False), (dict(heads=4, ld_q_token=128, ld_q_head=256), True),
                    (dict(heads=1, ld_q_token=128, k_out=1 << 51, ld_k_head=128, ld_k_token=1920), True),
                    (dict(heads=1, ld_q_token=128, k_out=1 << 51, ld_k_head=128, ld_k_token=2048), False)):
        status = _append(**dict(MANY, ld_token=36 * 128, **kw))
        assert (status == EINVAL and "rows of an output overlap" in _said()) if bad else \
            (status == EUNSUPPORTED and "too many" in _said()), (kw, _said())


def test_attention_output_over_its_queries():
    """Anywhere in their rows, not only at their beginning."""
    for out in (FAKE - 2 * 512 + 16, FAKE + 16, FAKE + 2 * 512, FAKE + 2 * (4 * 512 + 448), FAKE - 2 * (4 * 512 + 8)):
        assert _attend(out=out) == EINVAL and "overlap" in _said()
    wide = dict(ld_q_token=1024, ld_out=1024)
    assert _attend(out=FAKE + 2 * 504, **wide) == EINVAL and "overlap" in _said()
    assert _attend(out=FAKE - 2 * 520, **wide, ld_q_head=72) == EINVAL and "overlap" in _said()


@pytest.mark.parametrize("call", [_append, _attend, _compact])
def test_pages_whose_rows_pass_64_bits(call):
    for pages in (1 << 59, (1 << 59) + 1, 1 << 62):
        assert call(cache_pages=pages, cache_page_size=32) == EUNSUPPORTED and "int32" in _said()


def test_compactions_whose_waves_pass_64_bits():
    kw = dict(cache_kv_heads=16, cache_page_stride=16 * 32 * 64)
    for layers, batch in ((1 << 30, 1 << 30), (2 ** 31 - 1, 2 ** 31 - 1), (1 << 30, 1 << 29)):
        assert _compact(layers=layers, batch=batch, **kw) == EUNSUPPORTED and "too large" in _said()


@pytest.mark.parametrize("q", [_b(5, 8, 0), torch.zeros((), dtype=torch.bfloat16)])
def test_queries_without_elements_are_refused(q):
    with pytest.raises(TjkError):
        _py_attend(q=q, workspace=torch.zeros(64, dtype=torch.uint8))


def test_append_in_place_of_tokens_that_overlap():
    """A token's values that are the next one's queries may be read, but not while
    those are written."""
    one = dict(MANY, heads=2, ld_token=34 * 128 - 256, ld_q_token=256)
    assert _append(**one) == EUNSUPPORTED and "too many" in _said()
    place = dict(q_out=MANY["qkv"], ld_q_token=one["ld_token"])
    assert _append(**dict(one, **place)) == EINVAL and "overlap" in _said()
    keys = dict(k_out=MANY["qkv"] + 2 * 2 * 128, ld_k_token=one["ld_token"], ld_k_head=128, ld_q_token=256)
    assert _append(**dict(one, **keys)) == EINVAL and "overlap" in _said()
    for apart in (dict(one, **place), dict(one, **keys)):
        apart.update(ld_token=34 * 128, **{k: 34 * 128 for k in ("ld_q_token", "ld_k_token")})
        assert _append(**apart) == EUNSUPPORTED and "too many" in _said()
