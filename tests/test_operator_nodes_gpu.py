"""The engine's nodes over the 8-bit Linear, the head norms and the 4-bit cache,
each alone and as a decoder block's attention: projection, heads, cached
attention, output projection, recorded once and replayed as the sequence grows.
Every stage of the block is an output of the net and is checked against its
definition in 64 bits, given what the stage before it put out."""
import numpy as np
import pytest

import test_attention_q4_gpu as q4
import test_linear_i8_gpu as i8
import test_qk_norm_rope_gpu as rope
from helpers import draw, normal
from node_check import build_net, forward, pyvai

pytestmark = pytest.mark.gpu
F16, F32 = np.float16, np.float32


def rounded(w):
    """What a forward makes of a float weight [N, K]: integers and scales."""
    return i8.codes64(w)


@pytest.mark.parametrize("m, n, k, residual, epi, wdt", [(1, 48, 64, False, "NONE", F32), (9, 40, 100, True, "RELU", F16),
                                                         (33, 96, 130, True, "GELU_TANH", F32), (300, 256, 512, False, "SILU", F16)])
def test_linear_node(gpu, m, n, k, residual, epi, wdt):
    pv, rng = pyvai(), np.random.default_rng(m)
    w, b = draw(normal((n, k), k ** -0.5), rng, wdt), draw((n,), rng)
    net = build_net(lambda: pv.nodes.LinearNode(in_dim=k, out_dim=n, accept_residual=residual,
                                                epilogue=getattr(pv.Epilogue, epi), int8_weights=True),
                    ["in0", "residual"] if residual else ["in0"], {"weight": w, "bias": b})
    wq, ws = rounded(w)
    for rows in (m, m, m + 3):     # the second forward replays the first, the third records again
        fed = {"in0": draw((rows, k), rng)}
        if residual:
            fed["residual"] = draw((rows, n), rng)
        got = forward(net, fed)
        want, mag = i8.want64(fed["in0"], wq, ws, b, fed.get("residual"), epi)
        i8.check(got, want, mag, epi)
    assert net.node.plan == "i8" and net.record_count == 2
    net.node["weight"] = pv.Tensor.from_numpy(2 * w)      # a new weight is rounded again
    got = forward(net, fed)
    i8.check(got, *i8.want64(fed["in0"], wq, 2 * ws, b, fed.get("residual"), epi), epi)


def test_int8_linear_stays_apart_from_its_gate(gpu):
    """Linear -> GatedMul is one launch with fp16 weights; an 8-bit Linear keeps the two."""
    pv, rng = pyvai(), np.random.default_rng(1)
    k, h = 64, 48
    w = draw(normal((2 * h, k), 0.1), rng)

    class Net(pv.NeuralNet):
        def __init__(self):
            super().__init__()
            self.fc = pv.nodes.LinearNode(in_dim=k, out_dim=2 * h, int8_weights=True)
            self.gate = pv.nodes.GatedMulNode()
            self.input("x") - self.fc - self.gate - self.output("y")

    net = Net()
    net.fc["weight"] = pv.Tensor.from_numpy(w)
    x = draw((5, k), rng)
    got = net(x=pv.Tensor.from_numpy(x)).to_numpy()
    assert not net.fc.fused
    y, _ = i8.want64(x, *rounded(w))
    g, u = y[:, :h], y[:, h:]
    np.testing.assert_allclose(got, g / (1 + np.exp(-g)) * u, rtol=1e-4, atol=1e-5)


def test_refusals(gpu):
    pv = pyvai()
    net = pv.NeuralNet()   # the net that the nodes below belong to
    assert net.submit_count == 0
    with pytest.raises(RuntimeError, match="splitSize"):
        pv.nodes.LinearNode(in_dim=8, out_dim=8, split_size=64, int8_weights=True)
    with pytest.raises(RuntimeError, match="headDim <= 256"):
        pv.nodes.AttentionNode(4, 257, kv_cache_size=64, kv_cache_dtype=pv.Dtype.Q4)
    with pytest.raises(RuntimeError, match="rotDim"):
        pv.nodes.QkNormRopeNode(4, 64, rot_dim=66)
    with pytest.raises(RuntimeError, match="4-bit"):
        pv.Tensor.from_numpy(np.zeros(4, F32), pv.Dtype.Q4)
    with pytest.raises(RuntimeError, match="Q4"):
        pv.NeuralNet(o_default_dtype=pv.Dtype.Q4)

    class Net(pv.NeuralNet):
        def __init__(self):
            super().__init__()
            self.heads = pv.nodes.QkNormRopeNode(4, 64)
            self.input("x") - self.heads
            (self.heads / "Q") - self.output("q")

    with pytest.raises(RuntimeError, match="in0 must be"):
        Net()(x=pv.Tensor.from_numpy(np.zeros((3, 4 * 64), F32)))


@pytest.mark.parametrize("odt", ["F32", "F16"])
@pytest.mark.parametrize("d, hq, hkv, ring", [(64, 4, 2, False), (128, 8, 2, True), (72, 3, 3, False)])
def test_decoder_attention(gpu, d, hq, hkv, ring, odt):
    pv, rng = pyvai(), np.random.default_rng(d)
    dim, size = 96, 256
    row = (hq + 2 * hkv) * d
    counter = gpu.DeviceArray.from_numpy(np.zeros(1, np.uint32))

    class Net(pv.NeuralNet):
        def __init__(self):
            super().__init__(o_default_dtype=getattr(pv.Dtype, odt))
            self.qkv = pv.nodes.LinearNode(in_dim=dim, out_dim=row, int8_weights=True)
            self.heads = pv.nodes.QkNormRopeNode(hq, d, hkv, eps=1e-5, theta=500000.0)
            self.att = pv.nodes.AttentionNode(hq, d, hkv, kv_cache_size=size, kv_cache_dtype=pv.Dtype.Q4,
                                              kv_cache_ring=ring)
            self.input("x") - self.qkv - self.heads
            self.qkv - self.output("qkv")
            for slot in "QKV":
                (self.heads / slot) - (slot / self.att)
                (self.heads / slot) - self.output(slot)
            self.att - self.output("att")

    class Out(pv.NeuralNet):
        def __init__(self):
            super().__init__(o_default_dtype=getattr(pv.Dtype, odt))
            self.fc = pv.nodes.LinearNode(in_dim=hq * d, out_dim=dim, accept_residual=True, int8_weights=True)
            self.input("in0") - self.fc - self.output("out0")
            self.input("residual") - ("residual" / self.fc)

    net, out_net = Net(), Out()
    w, wo = draw(normal((row, dim), dim ** -0.5), rng, F16), draw(normal((dim, hq * d), 0.05), rng, F16)
    qw, kw = (1 + draw(normal((d,), 0.1), rng) for _ in range(2))
    net.qkv["weight"], out_net.fc["weight"] = pv.Tensor.from_numpy(w), pv.Tensor.from_numpy(wo)
    net.heads["q_weight"], net.heads["k_weight"] = pv.Tensor.from_numpy(qw), pv.Tensor.from_numpy(kw)
    net.att.set_causal_mask(1)
    net.att.set_kv_cache_counter(counter.ptr)
    net.heads.set_position_counter(counter.ptr)
    dt = F32 if odt == "F32" else F16
    rows, n = [np.zeros((hkv, 0, d)) for _ in range(2)], 0
    # a prompt, then tokens one by one, then a few at once (a ring wraps on the way)
    for tokens in (150, 1, 1, 1, 4, 90, 1, 1, 30, 1):
        if not ring and n + tokens > size:
            break
        x = draw((tokens, dim), rng, dt)
        gpu.check(gpu.lib().vai_memcpy_h2d(counter.ptr, np.array([n], np.uint32).ctypes.data, 4, None), "h2d")
        got = {s: t.to_numpy() for s, t in net(x=pv.Tensor.from_numpy(x)).items()}
        print(f"block d={d} at {n} + {tokens}", flush=True)
        i8.check(got["qkv"], *i8.want64(x, *rounded(w)), "NONE")
        pos = np.arange(n, n + tokens)[None]
        rope.check(tuple(got[s][None] for s in "QKV"),
                   *rope.want64(got["qkv"][None], hq, hkv, d, qw, kw, True, 1e-5, 0.0, "HALVES", 0, 500000.0, pos))
        rows = [np.concatenate([r, q4.stored(got[s])], 1) for r, s in zip(rows, "KV")]
        first = max(0, n + tokens - size) if ring else 0
        see = q4.visible(n, tokens, tokens, first, size - tokens + 1 if ring else 0)
        want, tol = q4.attend(got["Q"], *(r[:, first:] for r in rows), see, dt == F32)
        q4.check(got["att"], want, tol)
        att = got["att"].reshape(tokens, hq * d)
        y = out_net(in0=pv.Tensor.from_numpy(att), residual=pv.Tensor.from_numpy(x)).to_numpy()
        want, mag = i8.want64(att, *rounded(wo), residual=x)
        i8.check(y, want, mag, "NONE")
        n += tokens
    assert net.record_count < net.submit_count    # single tokens replay
