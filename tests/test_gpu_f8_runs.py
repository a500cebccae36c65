"""The 8-bit operators as they are used: one after another through a layer, in
a captured graph, on several streams at once; and the calls at the edges of
what they take (nothing to add up, NaN operands, buffers past 2 GB)."""

import pytest
import torch

from tjkernels import ops
from tjkernels.ops import EPI_BIAS_GELU, F8

from test_gpu_f8 import Y_ERR, _blocks, _check_quantised, _gelu, _gelu_err, _gen, _product

pytestmark = pytest.mark.gpu


def _value(q, scales, block_rows):
    """The 64-bit matrix that q and scales stand for."""
    s = scales.double().cpu().repeat_interleave(block_rows, 0)[:q.shape[0]]
    return q.float().double().cpu() * s.repeat_interleave(128, 1)[:, :q.shape[1]]


class Layer:
    """Feed-forward half of a pre-norm layer on 8-bit operands: x += delta;
    h = norm(x); u = gelu(h W1 + b1) in e4m3; delta = u W2 + b2."""

    def __init__(self, t, d, f, device, seed=0):
        g = _gen(seed)

        def weight(rows, cols):
            w = (torch.randn(rows, cols, generator=g) / cols ** 0.5).to(device)
            q = torch.empty(rows, cols, dtype=F8, device=device)
            s = torch.empty(_blocks(rows), _blocks(cols), device=device)
            ops.quantize_f8(w, q, s, block_rows=128)
            return q, s

        self.w1, self.w2 = weight(f, d), weight(d, f)
        self.b1 = torch.randn(f, generator=g).to(device)
        self.b2 = torch.randn(d, generator=g).bfloat16().to(device)
        self.gamma = (1 + 0.1 * torch.randn(d, generator=g)).to(device)
        self.x = torch.randn(t, d, generator=g).to(device)
        self.delta = torch.randn(t, d, generator=g).bfloat16().to(device)
        self.h = torch.empty(t, d, dtype=F8, device=device), torch.empty(t, _blocks(d), device=device)
        self.u = torch.empty(t, f, dtype=F8, device=device), torch.empty(t, _blocks(f), device=device)

    def run(self):
        (h, hs), (u, us) = self.h, self.u
        ops.add_rmsnorm(self.x, self.delta, self.gamma, 1e-5, h, res_out=self.x, scales=hs)
        ops.gemm_f8(h, hs, *self.w1, self.b1, u, EPI_BIAS_GELU, out_scales=us)
        ops.gemm_f8(u, us, *self.w2, self.b2, self.delta)

    def state(self):
        return [t.view(torch.uint8).clone() if t.dtype == F8 else t.clone()
                for t in (self.x, *self.h, *self.u, self.delta)]


def _same(a, b):
    return all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("t,d,f", [(1, 256, 1024), (37, 272, 1040), (300, 512, 2048)])
def test_a_layer_of_them(device, t, d, f):
    """Twice through the layer; each operator's result against 64 bits of what
    it was given."""
    layer = Layer(t, d, f, device, seed=t)
    w1, w2 = _value(*layer.w1, 128), _value(*layer.w2, 128)
    for _ in range(2):
        x0, d0 = layer.x.cpu(), layer.delta.float().cpu()
        layer.run()
        torch.cuda.synchronize()
        x = x0 + d0
        assert torch.equal(layer.x.cpu(), x)
        x = x.double()
        y = x / (x.square().mean(1, keepdim=True) + 1e-5).sqrt() * layer.gamma.double().cpu()
        _check_quantised(*layer.h, y, 1, Y_ERR * y.abs())
        v, _, err = _product(_value(*layer.h, 1), w1, layer.b1.double().cpu())
        err, v = _gelu_err(v, err), _gelu(v)
        _check_quantised(*layer.u, v, 1, err)
        v, err, _ = _product(_value(*layer.u, 1), w2, layer.b2.double().cpu())
        got = layer.delta.double().cpu()
        assert ((got - v).abs() <= err + 2.0 ** -8 * (v.abs() + err) + 2.0 ** -25).all()


@pytest.mark.parametrize("t", [3, 130])
def test_captured(device, t):
    """A captured layer, replayed with other inputs between eager runs of
    another one on the default stream, gives what eager calls give, bit by bit."""
    eager, captured, other = (Layer(t, 256, 1024, device, seed=5) for _ in range(3))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        captured.run()  # loads the code
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured.run()
        captured.run()
    g = _gen(9)
    for _ in range(4):
        x = torch.randn(t, 256, generator=g).to(device)
        for layer in (eager, captured):
            layer.x.copy_(x)
            layer.delta.copy_(x.flip(0))
        graph.replay()
        other.run()
        eager.run()
        eager.run()
        torch.cuda.synchronize()
        assert _same(eager.state(), captured.state())


def test_two_graphs_at_once(device):
    """Two captured layers share no memory of the library's own."""
    layers = [Layer(130, 256, 1024, device, seed=s) for s in (1, 2)]
    want, graphs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    starts = [(l.x.clone(), l.delta.clone()) for l in layers]
    for l in layers:
        for _ in range(8):
            l.run()
        torch.cuda.synchronize()
        want.append(l.state())
    for l, s in zip(layers, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            for _ in range(8):
                l.run()
        graphs.append(graph)
    for _ in range(3):
        for l, (x, delta) in zip(layers, starts):
            l.x.copy_(x)
            l.delta.copy_(delta)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert all(_same(l.state(), w) for l, w in zip(layers, want))


def test_streams(device):
    """Calls run on the current stream, in its order, also when tensors were
    made on another one; two streams at once do not disturb each other."""
    layers = [Layer(200, 512, 2048, device, seed=s) for s in (3, 4)]
    alone = [Layer(200, 512, 2048, device, seed=s) for s in (3, 4)]
    torch.cuda.synchronize()
    for layer in alone:
        for _ in range(20):
            layer.run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in layers]
    for _ in range(20):
        for layer, s in zip(layers, streams):
            with torch.cuda.stream(s):
                layer.run()
    torch.cuda.synchronize()
    assert all(_same(a.state(), b.state()) for a, b in zip(alone, layers))


@pytest.mark.parametrize("plan", range(9))
def test_no_depth(device, plan):
    """K = 0: the epilogue of the bias alone, and no operand is read."""
    m, n = 37, 132
    bias = torch.randn(n, generator=_gen(1))
    a, a_s = torch.empty(m, 0, dtype=F8, device=device), torch.empty(m, 0, device=device)
    w, w_s = torch.empty(n, 0, dtype=F8, device=device), torch.empty(2, 0, device=device)
    out = torch.full((m, n), 7.0, dtype=torch.bfloat16, device=device)
    ops.gemm_f8(a, a_s, w, w_s, bias.bfloat16().to(device), out, plan=plan)
    assert torch.equal(out.cpu(), bias.bfloat16().expand(m, n))
    ops.gemm_f8(a, a_s, w, w_s, None, out, plan=plan)
    assert (out == 0).all()
    if plan < 3:
        q, s = torch.empty(m, n, dtype=F8, device=device), torch.empty(m, 2, device=device)
        ops.gemm_f8(a, a_s, w, w_s, bias.to(device), q, out_scales=s, plan=plan)
        y = bias.double().expand(m, n)
        _check_quantised(q, s, y, 1, torch.zeros(m, n, dtype=torch.double))


def test_nothing_to_multiply(device):
    w, w_s = torch.zeros(128, 256, dtype=F8, device=device), torch.ones(1, 2, device=device)
    out = torch.empty(0, 128, dtype=torch.bfloat16, device=device)
    ops.gemm_f8(torch.empty(0, 256, dtype=F8, device=device), torch.empty(0, 2, device=device), w, w_s, None, out)
    ops.add_rmsnorm(torch.empty(0, 128, device=device), None, torch.ones(128, device=device), 1e-5,
                    torch.empty(0, 128, dtype=F8, device=device), scales=torch.empty(0, 1, device=device))
    torch.cuda.synchronize()


@pytest.mark.parametrize("plan", range(-1, 9))
def test_nan_stays_in_its_row_and_column(device, plan):
    """A NaN in a row of a (or its scale) makes that row of the output NaN, one
    in a row of w that column, and nothing else differs."""
    m, n, k = 70, 140, 400
    g = _gen(2)
    a = (torch.randn(m, k, generator=g) * 50).to(F8)
    w = (torch.randn(n, k, generator=g) * 50).to(F8)
    a_s, w_s = torch.rand(m, 4, generator=g) + 0.1, torch.rand(2, 4, generator=g) + 0.1
    args = [t.to(device) for t in (a, a_s, w, w_s)]
    bad_a, bad_w, bad_s = a.clone(), w.clone(), a_s.clone()
    bad_a.view(torch.uint8)[33, 399] = 0x7F
    bad_w.view(torch.uint8)[101, 0] = 0xFF
    bad_s[5, 3] = float("nan")
    bad = [t.to(device) for t in (bad_a, bad_s, bad_w, w_s)]
    want, got = (torch.empty(m, n, dtype=torch.bfloat16, device=device) for _ in range(2))
    ops.gemm_f8(*args, None, want, plan=plan)
    ops.gemm_f8(*bad, None, got, plan=plan)
    assert torch.isnan(got[33]).all() and torch.isnan(got[5]).all() and torch.isnan(got[:, 101]).all()
    got[33], got[5], got[:, 101] = want[33], want[5], want[:, 101]
    assert torch.equal(want, got)
    if plan < 3:
        outs = []
        for s in (args, bad):
            q, s_out = torch.empty(m, n, dtype=F8, device=device), torch.empty(m, 2, device=device)
            ops.gemm_f8(*s, None, q, out_scales=s_out, plan=plan)
            outs.append((q.float(), s_out))
        (q0, s0), (q1, s1) = outs
        assert torch.isnan(q1[33]).all() and torch.isnan(q1[5]).all() and torch.isnan(q1[:, 101]).all()
        keep = torch.ones(m, dtype=torch.bool, device=device)
        keep[33] = keep[5] = False
        # column 101's block takes its scale from the other columns
        assert torch.equal(s1[keep, 1], s0[keep, 1]) and torch.isfinite(s1[keep]).all()
        assert torch.equal(q1[keep][:, 128:], q0[keep][:, 128:])


def test_one_tensor_for_both_operands(device):
    """x x^T of one tensor, with the scales of 128 equal rows."""
    m, k = 128, 640
    x = (torch.randn(m, k, generator=_gen(4)) * 60).to(F8)
    s = torch.rand(1, 5, generator=_gen(5)) + 0.5
    q, a_s, w_s = x.to(device), s.expand(m, 5).contiguous().to(device), s.to(device)
    out = torch.empty(m, m, dtype=torch.bfloat16, device=device)
    ops.gemm_f8(q, a_s, q, w_s, None, out)
    val = _value(x, s.expand(m, 5), 1)
    v, err, _ = _product(val, val, None)
    assert ((out.double().cpu() - v).abs() <= err + 2.0 ** -8 * (v.abs() + err)).all()
    again = torch.empty_like(out)
    ops.gemm_f8(q, a_s, q, w_s, None, again)
    assert torch.equal(out, again)


@pytest.mark.parametrize("stride", [1, 7, 4096])
def test_one_row_of_any_stride(device, stride):
    """A matrix of one row may have any row stride."""
    n = 256
    x = torch.randn(1, n, generator=_gen(6)).to(device)
    odd = x.as_strided((1, n), (stride, 1))
    q, s = torch.empty(2, 1, n, dtype=F8, device=device), torch.empty(2, 1, 2, device=device)
    ops.quantize_f8(x, q[0], s[0])
    ops.quantize_f8(odd, q[1].as_strided((1, n), (stride, 1), q[1].storage_offset()), s[1])
    assert torch.equal(q[0].view(torch.uint8), q[1].view(torch.uint8)) and torch.equal(s[0], s[1])


@pytest.mark.parametrize("plan", [-1, 0, 3])
def test_gemm_past_2_gb(device, plan):
    """An output and an operand whose bytes do not fit 32 bits: rows at the
    far end are right, and the row behind the last is left alone."""
    m, n, k = 36000, 65536, 128
    g = _gen(7)
    a = torch.zeros(m, 65536, dtype=F8, device=device)[:, 256:256 + k]  # rows 64 KB apart
    rows = torch.tensor([0, 1, 16383, 16384, 32767, 32768, 35871, 35999])
    vals = (torch.randn(len(rows), k, generator=g) * 60).to(F8)
    a.view(torch.uint8)[rows.to(device)] = vals.view(torch.uint8).to(device)
    w = (torch.randn(n, k, generator=g) * 60).to(F8)
    a_s, w_s = torch.ones(m, 1), torch.rand(n // 128, 1, generator=g) + 0.1
    whole = torch.full((m + 1, n), 3.0, dtype=torch.bfloat16, device=device)
    ops.gemm_f8(a, a_s.to(device), w.to(device), w_s.to(device), None, whole[:m], plan=plan)
    v, err, _ = _product(vals.float().double(), _value(w, w_s, 128), None)
    got = whole[rows.to(device)].double().cpu()
    assert ((got - v).abs() <= err + 2.0 ** -8 * (v.abs() + err)).all()
    rest = torch.ones(m, dtype=torch.bool, device=device)
    rest[rows.to(device)] = False
    assert all((part == 0).all() for part in whole[:m][rest].split(4096))
    assert (whole[m] == 3.0).all()


def test_rows_past_2_gb(device):
    """The norm and the quantisation of a matrix of more than 2^31 elements."""
    m, n = 270000, 8192
    x = torch.zeros(m, n, dtype=torch.bfloat16, device=device)
    rows = torch.tensor([0, 131071, 131072, 262143, 262144, m - 1])
    vals = torch.randn(len(rows), n, generator=_gen(8)).bfloat16()
    x[rows.to(device)] = vals.to(device)
    q = torch.empty(m, n, dtype=F8, device=device)
    s = torch.empty(m, n // 128, device=device)
    ops.quantize_f8(x, q, s)
    pick = rows.to(device)
    y = vals.double()
    _check_quantised(q[pick], s[pick], y, 1, torch.zeros_like(y))
    zero = torch.ones(m, dtype=torch.bool, device=device)
    zero[pick] = False
    assert (s[zero] == 2.0 ** -126).all()
    sq = torch.empty(-(-m // 128), n // 128, device=device)
    ops.quantize_f8(x, q, sq, block_rows=128)
    blocks = (rows // 128).to(device)
    for i, r in enumerate(rows.tolist()):  # each in a block of its own: 128 rows apart or more, or not at all
        if sum(o // 128 == r // 128 for o in rows.tolist()) == 1:
            _check_quantised(q[r:r + 1], sq[blocks[i]:blocks[i] + 1], y[i:i + 1], 1, torch.zeros_like(y[i:i + 1]))
    gamma = torch.ones(n, device=device)
    ops.add_rmsnorm(x, x, gamma, 1e-5, q, res_out=x, scales=s)
    x64 = (2 * vals.float()).double()
    y = x64 / (x64.square().mean(1, keepdim=True) + 1e-5).sqrt()
    _check_quantised(q[pick], s[pick], y, 1, Y_ERR * y.abs())
    assert torch.equal(x[pick].cpu(), 2 * vals)


def test_other_tensors_refused(device):
    """What the calls refuse of device tensors."""
    x = torch.zeros(4, 256, device=device)
    q, s = torch.zeros(4, 256, dtype=F8, device=device), torch.zeros(4, 2, device=device)
    with pytest.raises(ops.TjkError, match="tensors on"):
        ops.quantize_f8(x, q.cpu(), s)
    with pytest.raises(ops.TjkError, match="tensors on"):
        ops.add_rmsnorm(x, None, torch.ones(256), 1e-5, q, scales=s)
    with pytest.raises(ops.TjkError, match="misaligned"):
        ops.quantize_f8(torch.zeros(4, 260, device=device).flatten()[1:1025].view(4, 256), q, s)
    with pytest.raises(ops.TjkError, match="leading"):
        ops.quantize_f8(x[:1].expand(4, 256), q, s)
    with pytest.raises(ops.TjkError, match="alias"):
        ops.add_rmsnorm(x, None, torch.ones(256, device=device), 1e-5, q, scales=s,
                        res_out=x.view(torch.bfloat16)[:, :256])
    assert (q.float() == 0).all() and (s == 0).all() and (x == 0).all()
