"""Two layers over their pages, the logits and the check of drafts in one recorded net, which then advances its own
counts. Every stage is checked against its definition in 64 bits, given what the stage before it put out."""
import numpy as np
import pytest

import test_paged_attention_gpu as att
import test_qk_norm_rope_gpu as rope
import test_verify_drafts_gpu as ver
from helpers import draw, normal
from node_check import pyvai
from paged import Batch, F16, F32
from test_paged_nodes_gpu import set_pages

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("odt", ["F32", "F16"])
def test_layers_and_check_in_one_net(gpu, odt, with_draft):
    pv, rng = pyvai(), np.random.default_rng(7)
    d, vocab, n_seq, rows, page = 64, 700, 3, 12, 16        # (one head: its values are the next Linear's rows)
    dt = F32 if odt == "F32" else F16
    D = gpu.DeviceArray.from_numpy
    layers = [Batch(gpu, rng, [1] * n_seq, [199] * n_seq, 1, d, page, F16) for _ in range(2)]

    class Net(pv.NeuralNet):
        def __init__(self):
            super().__init__(o_default_dtype=getattr(pv.Dtype, odt))
            self.layers = []
            last = self.input("x")
            for i in range(2):
                qkv, heads = pv.nodes.LinearNode(in_dim=d, out_dim=3 * d), pv.nodes.PagedAppendNode(1, d, norm=False)
                attention = pv.nodes.PagedAttentionNode(1, d, max_new=8)
                last - qkv - heads
                (heads / "Q") - ("Q" / attention)
                qkv - self.output(f"qkv{i}")
                (heads / "Q") - self.output(f"Q{i}")
                attention - self.output(f"att{i}")
                self.layers.append((qkv, heads, attention))
                last = attention
            self.head, self.check = pv.nodes.LinearNode(in_dim=d, out_dim=vocab), pv.nodes.VerifyDraftsNode()
            last - self.head
            self.head - self.output("logits")
            self.head - ("target" / self.check)
            if with_draft:
                self.input("draft") - ("draft" / self.check)

    net = Net()
    held = [3, 0, 40]
    for b, (qkv, heads, attention) in zip(layers, net.layers):
        for s, h in enumerate(held):      # what the pages hold before
            b.store(s, *(draw((h, 1, d), rng, F32).astype(F16) for _ in range(2)))
        b.held, b.new = list(held), [4] * n_seq
        b.starts = np.array([0, 4, 8, 12], np.uint32)
        b.upload()
        b.upload_tables()
        qkv["weight"] = pv.Tensor.from_numpy(draw(normal((3 * d, d), 3 * d ** -0.5), rng, F16))
    net.head["weight"] = pv.Tensor.from_numpy(draw(normal((vocab, d), 3 * d ** -0.5), rng, F16))
    one = layers[0]
    layers[1].d_start, layers[1].d_counts = one.d_start, one.d_counts
    for b, (_, heads, attention) in zip(layers, net.layers):
        for node in (heads, attention):
            set_pages(pv, node, b)
    dev = {n: D(np.zeros(k, t)) for n, k, t in (("tokens", rows, np.uint32), ("uniform", rows, F32), ("out", rows, np.uint32),
                                                ("accepted", n_seq, np.uint32), ("temp", n_seq, F32))}
    h2d = lambda dst, a: gpu.check(gpu.lib().vai_memcpy_h2d(dst.ptr, a.ctypes.data, a.nbytes, None), "h2d")  # noqa: E731
    temps = np.array([0.9, 0.0, 1.3], F32)
    h2d(dev["temp"], temps)
    net.check.set_batch(n_seq, one.d_start.ptr, dev["tokens"].ptr, dev["uniform"].ptr, dev["out"].ptr, dev["accepted"].ptr,
                        temperature=dev["temp"].ptr, counts=one.d_counts.ptr, new_counts=one.d_counts.ptr)
    for step, starts in enumerate(([0, 4, 8, 12], [0, 1, 2, 12], [0, 6, 6, 9], [0, 4, 8, 12])):
        starts = np.array(starts, np.uint32)
        h2d(one.d_start, starts)
        draft = (3 * draw((rows, 1, 1, vocab), rng, F32)).astype(dt)     # (each layer adds its heads' axis)
        tokens, u = rng.integers(0, vocab, rows).astype(np.uint32), rng.uniform(0, 1, rows).astype(F32)
        if step % 2:
            u[:] *= 1e-3                  # drafts of some probability are kept
        h2d(dev["tokens"], tokens)
        h2d(dev["uniform"], u)
        fed = {"x": pv.Tensor.from_numpy(draw((rows, d), rng, dt))}
        if with_draft:
            fed["draft"] = pv.Tensor.from_numpy(draft)
        print(f"one net step {step} held={held} starts={list(starts)} draft={with_draft}", flush=True)
        got = {s: t.to_numpy() for s, t in net(**fed).items()}
        got = {s: x.reshape(rows, 1, d) if s[0] in "Qa" else x.reshape(rows, -1) for s, x in got.items()}
        net.sync()
        for i, b in enumerate(layers):
            b.starts, b.new, b.held = starts, list(np.diff(starts.astype(int))), list(held)
            k_now, v_now = b.download()
            b.K, b.V = [], []
            for s, n in enumerate(b.new):
                pos, at = np.arange(held[s] + n), int(starts[s])
                pg, slot = b.table[s, pos // page], pos % page
                b.K.append(k_now[pg, :, slot])
                b.V.append(v_now[pg, :, slot])
                if n == 0:
                    continue
                want, mag = rope.want64(got[f"qkv{i}"][None, at:at + n], 1, 1, d, None, None, False, 1e-6, 0.0, "HALVES", d,
                                        10000.0, pos[held[s]:][None])
                new = tuple(z[-1][held[s]:].transpose(1, 0, 2)[None] for z in (b.K, b.V))
                rope.check((got[f"Q{i}"][at:at + n].transpose(1, 0, 2)[None], *new), want, mag)
            att.check(b, got[f"Q{i}"], got[f"att{i}"], dt)
        want, acc = ver.verify(got["logits"], draft.reshape(rows, vocab) if with_draft else None, tokens, u,
                               starts, temps)
        np.testing.assert_array_equal(dev["out"].numpy()[:starts[-1]], want[:int(starts[-1])])
        np.testing.assert_array_equal(dev["accepted"].numpy(), [a or 0 for a in acc])
        held = [h if a is None else h + a + 1 for h, a in zip(held, acc)]
        np.testing.assert_array_equal(one.d_counts.numpy(), held)     # advanced by the net itself
    assert net.record_count == 1 and net.submit_count == 4
