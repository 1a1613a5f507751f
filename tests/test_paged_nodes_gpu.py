"""The engine's nodes over a KV cache in pages: refusals, and a decoder block's
attention, its logits and the check of drafts in recorded nets, step after step. Every
stage is checked against its definition in 64 bits, given what the stage before it
put out; the lengths advance on the device."""
import numpy as np
import pytest

import test_paged_attention_gpu as att
import test_qk_norm_rope_gpu as rope
import test_verify_drafts_gpu as ver
from helpers import draw, normal
from node_check import pyvai
from paged import Batch, F16, F32

pytestmark = pytest.mark.gpu


def set_pages(pv, node, b):
    node.set_pages(b.d_k.ptr, b.d_v.ptr, b.d_table.ptr, b.d_start.ptr, b.d_counts.ptr, len(b.new), b.num_pages, b.page,
                   b.table.shape[1], pv.Dtype.F16 if b.dt == F16 else pv.Dtype.F32,
                   page_stride=b.stride if b.gap is not None else 0)


def test_refusals(gpu):
    pv = pyvai()
    net = pv.NeuralNet()
    assert net.submit_count == 0
    with pytest.raises(RuntimeError, match="rotDim"):
        pv.nodes.PagedAppendNode(4, 64, rot_dim=66)
    with pytest.raises(RuntimeError, match="at most 256"):
        pv.nodes.PagedAttentionNode(4, 257)
    with pytest.raises(RuntimeError, match="multiple of numKVHeads"):
        pv.nodes.PagedAttentionNode(4, 64, 3)
    with pytest.raises(ValueError, match="F32 or F16"):
        pv.nodes.PagedAttentionNode(4, 64).set_pages(1, 1, 1, 1, 1, 1, 1, 16, 1, pv.Dtype.Q4)

    def one(make, slot, out=None):
        class Net(pv.NeuralNet):
            def __init__(self):
                super().__init__()
                self.node = make()
                self.input("x") - (slot / self.node)
                if out:
                    (self.node / out) - self.output("y")
                else:
                    self.fc = pv.nodes.GatedMulNode()
                    self.input("z") - self.fc - self.output("y")
        return Net()

    x = pv.Tensor.from_numpy(np.zeros((3, 4, 64), F32))
    with pytest.raises(RuntimeError, match="in0 must be"):
        one(lambda: pv.nodes.PagedAppendNode(4, 64), "in0", "Q")(x=x)
    with pytest.raises(RuntimeError, match="setPages"):
        one(lambda: pv.nodes.PagedAppendNode(2, 16), "in0", "Q")(x=pv.Tensor.from_numpy(np.zeros((3, 96), F32)))
    with pytest.raises(RuntimeError, match="Q must be"):
        one(lambda: pv.nodes.PagedAttentionNode(3, 64), "Q", "out0")(x=x)
    with pytest.raises(RuntimeError, match="setPages"):
        one(lambda: pv.nodes.PagedAttentionNode(4, 64), "Q", "out0")(x=x)
    with pytest.raises(RuntimeError, match="setBatch"):
        one(lambda: pv.nodes.VerifyDraftsNode(), "target")(x=x, z=pv.Tensor.from_numpy(np.zeros((2, 4), F32)))
    # what the launch refuses comes out of the forward
    node = one(lambda: pv.nodes.PagedAttentionNode(4, 64), "Q", "out0")
    node.node.set_pages(256, 256, 256, 256, 256, 5000, 4, 16, 4, pv.Dtype.F16)
    with pytest.raises(RuntimeError):
        node(x=x)


@pytest.mark.parametrize("odt, pdt, d, hq, hkv, page", [("F32", F16, 64, 4, 2, 16), ("F16", F16, 128, 8, 2, 32),
                                                        ("F32", F32, 50, 3, 3, 12)])
def test_speculative_steps(gpu, odt, pdt, d, hq, hkv, page):
    pv, rng = pyvai(), np.random.default_rng(d)
    dim, vocab, n_seq, rows = 96, 700, 3, 12
    row = (hq + 2 * hkv) * d
    dt = F32 if odt == "F32" else F16
    D = gpu.DeviceArray.from_numpy
    # room for 200 positions a sequence, page by page from one pool
    b = Batch(gpu, rng, [1] * n_seq, [199] * n_seq, hkv, d, page, pdt, gap=8 * 4)
    b.upload()

    class Net(pv.NeuralNet):
        def __init__(self):
            super().__init__(o_default_dtype=getattr(pv.Dtype, odt))
            self.qkv = pv.nodes.LinearNode(in_dim=dim, out_dim=row)
            self.heads = pv.nodes.PagedAppendNode(hq, d, hkv, eps=1e-5, theta=500000.0, rot_dim=d // 4 * 2)
            self.att = pv.nodes.PagedAttentionNode(hq, d, hkv)
            self.input("x") - self.qkv - self.heads
            self.qkv - self.output("qkv")
            (self.heads / "Q") - ("Q" / self.att)
            (self.heads / "Q") - self.output("Q")
            self.att - self.output("att")

    class Head(pv.NeuralNet):
        def __init__(self):
            super().__init__(o_default_dtype=getattr(pv.Dtype, odt))
            self.head = pv.nodes.LinearNode(in_dim=hq * d, out_dim=vocab)
            self.check = pv.nodes.VerifyDraftsNode()
            self.input("h") - self.head
            self.head - self.output("logits")
            self.head - ("target" / self.check)
            self.input("draft") - ("draft" / self.check)

    net, head = Net(), Head()
    qw, kw = (1 + draw(normal((d,), 0.1), rng) for _ in range(2))
    net.qkv["weight"] = pv.Tensor.from_numpy(draw(normal((row, dim), dim ** -0.5), rng, F16))
    wh = draw(normal((vocab, hq * d), 3 * (hq * d) ** -0.5), rng, F16)
    head.head["weight"] = pv.Tensor.from_numpy(wh)
    net.heads["q_weight"], net.heads["k_weight"] = pv.Tensor.from_numpy(qw), pv.Tensor.from_numpy(kw)
    held = [3, 0, 40]
    b.held = list(held)
    b.new = [4, 4, 4]
    b.starts = np.array([0, 4, 8, 12], np.uint32)
    for s, h in enumerate(held):      # what the pages hold before
        k, v = (draw((h, hkv, d), rng, F32).astype(pdt) for _ in range(2))
        b.store(s, k, v)
    b.upload()
    b.upload_tables()
    dev = {n: D(np.zeros(k, t)) for n, k, t in (("tokens", rows, np.uint32), ("uniform", rows, F32), ("out", rows, np.uint32),
                                                ("accepted", n_seq, np.uint32), ("temp", n_seq, F32))}
    h2d = lambda dst, a: gpu.check(gpu.lib().vai_memcpy_h2d(dst.ptr, a.ctypes.data, a.nbytes, None), "h2d")  # noqa: E731
    temps = np.array([0.9, 0.0, 1.3], F32)
    h2d(dev["temp"], temps)
    for node in (net.heads, net.att):
        set_pages(pv, node, b)
    head.check.set_batch(n_seq, b.d_start.ptr, dev["tokens"].ptr, dev["uniform"].ptr, dev["out"].ptr, dev["accepted"].ptr,
                        temperature=dev["temp"].ptr, counts=b.d_counts.ptr, new_counts=b.d_counts.ptr)
    for step, starts in enumerate(([0, 4, 8, 12], [0, 4, 8, 12], [0, 1, 2, 12], [0, 6, 6, 9], [0, 4, 8, 12])):
        starts = np.array(starts, np.uint32)
        b.starts, b.new, b.held = starts, list(np.diff(starts.astype(int))), list(held)
        h2d(b.d_start, starts)
        x = draw((rows, dim), rng, dt)
        was = b.download()
        got = {s: t.to_numpy() for s, t in net(x=pv.Tensor.from_numpy(x)).items()}
        hid = np.nan_to_num(got["att"].reshape(rows, hq * d))     # (rows of no sequence hold anything)
        draft = (3 * draw((rows, vocab), rng, F32)).astype(dt)
        tokens, u = rng.integers(0, vocab, rows).astype(np.uint32), rng.uniform(0, 1, rows).astype(F32)
        if step % 2:                  # a model that drafts what the target wants
            draft = (hid.astype(F32) @ wh.astype(F32).T).astype(dt)
            tokens[1:] = draft[:-1].argmax(-1)
        h2d(dev["tokens"], tokens)
        h2d(dev["uniform"], u)
        got["logits"] = head(h=pv.Tensor.from_numpy(hid), draft=pv.Tensor.from_numpy(draft)).to_numpy()
        head.sync()
        print(f"paged step {step} d={d} held={held} starts={list(starts)}", flush=True)
        k_now, v_now = b.download()
        b.K, b.V = [], []
        for s, n in enumerate(b.new):
            pos = np.arange(held[s] + n)
            pg, slot = b.table[s, pos // page], pos % page
            K, V = k_now[pg, :, slot], v_now[pg, :, slot]
            b.K.append(K)
            b.V.append(V)
            old = pos < held[s]
            np.testing.assert_array_equal(K[old], was[0][pg, :, slot][old])
            if n == 0:
                continue
            at = int(starts[s])
            want, mag = rope.want64(got["qkv"][None, at:at + n], hq, hkv, d, qw, kw, True, 1e-5, 0.0, "HALVES", d // 4 * 2,
                                    500000.0, pos[~old][None])
            new = tuple(z[~old].transpose(1, 0, 2)[None] for z in (K, V))
            rope.check((got["Q"][at:at + n].transpose(1, 0, 2)[None], *new), want, mag)
        att.check(b, got["Q"], got["att"], dt)
        want, acc = ver.verify(got["logits"], draft, tokens, u, starts, temps)
        np.testing.assert_array_equal(dev["out"].numpy()[:starts[-1]], want[:int(starts[-1])])
        np.testing.assert_array_equal(dev["accepted"].numpy(), [a or 0 for a in acc])
        held = [h if a is None else h + a + 1 for h, a in zip(held, acc)]
        np.testing.assert_array_equal(b.d_counts.numpy(), held)     # advanced on the device
    assert net.record_count == head.record_count == 1 and net.submit_count == 5
