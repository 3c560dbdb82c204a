"""A decode layer over the 8-bit cache, as a program would run it: prompts
prefilled in a context (bf16 pages), their rows moved into an 8-bit pool under
the same page ids, then steps of projection GEMV -> rotary (q and k in place in
the projection row) -> write -> attention with the row's gate -> output GEMV.

Checked per step: the rows against those that qc_attn_decode appends for the
same projections, the attention against 64 bits over the values read back, and
its distance from qc_attn_decode's output against what the quantisation can do:
a code is off by at most half a scale, at most u / 127 for a block whose largest
magnitude is u (127 scale <= 2 u), and a block that is rescaled once more by as
much again, so |dk| <= 2 u_k / 127 and |dv| <= 2 u_v / 127; a score moves by at
most d = scale sum|q| max(u_k) 2 / 127, a weight by a factor within e^(+-2d), and
an output by (e^(2d) - 1) sum p|v| + max(u_v) 2 / 127, times the gate (< 1), plus
the two roundings to bf16 and the bf16 kernel's own 1e-5.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from gpu_util import dev, empty_u16, host_u16  # noqa: E402
from test_gpu_bfp8 import assert_gemv_close  # noqa: E402
from test_gpu_kv8 import check_attention, i32  # noqa: E402

H, KV, D, HID, OUT = 16, 4, 256, 512, 256


def bf(t):
    return t.view(torch.bfloat16)


class Layer:
    """Weights, an 8-bit pool and the step's buffers for n sequences."""

    def __init__(self, qcache, synth, oracle, n, pages, width, q_norm, k_norm):
        self.qc, self.n, self.width = qcache, n, width
        self.win, self.wout = qcache.Bfp8Matrix(10240, HID), qcache.Bfp8Matrix(OUT, 4096)
        self.win.pack_bf16(dev(synth.bfp8_weights(901, 10240, HID, std=0.044, edges=False)).data_ptr())
        wo = synth.bfp8_weights(902, OUT, 4096, edges=False)
        self.wout.pack_bf16(dev(wo).data_ptr())
        self.packed_out = oracle.bfp8_pack(wo)
        self.pool = torch.zeros(pages * qcache.kv8_page_bytes(KV, D), dtype=torch.uint8, device="cuda")
        self.cache = qcache.Kv8Cache(self.pool.data_ptr(), pages, KV, D)
        self.rope = qcache.Rope(64)
        self.qn, self.kn = dev(q_norm), dev(k_norm)
        self.table = torch.zeros(n, width, dtype=torch.int32, device="cuda")
        self.pos, self.len = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in "pl")
        self.x = empty_u16(n, HID)
        self.proj, self.out, self.y = empty_u16(n, 10240), empty_u16(n, 4096), empty_u16(n, OUT)
        self.ws = torch.empty(self.cache.attn_workspace_bytes(n, H), dtype=torch.uint8, device="cuda")

    def project(self, st=0):
        self.win.gemv(self.x.data_ptr(), self.n, self.proj.data_ptr(), st)

    def attend(self, st=0):
        """Rotary, write, attention, output projection of the projected rows."""
        p, n = self.proj.data_ptr(), self.n
        part = self.qc.RopePart
        self.rope.apply(D, self.pos.data_ptr(), n,
                        [part(p, p, H, 10240, 512, 10240, 512, self.qn.data_ptr()),
                         part(p + 2 * 8192, p + 2 * 8192, KV, 10240, 256, 10240, 256, self.kn.data_ptr())], 1e-6, st)
        self.cache.write(self.table.data_ptr(), self.width, self.pos.data_ptr(), 0, n, n, p + 2 * 8192, 10240,
                         p + 2 * 9216, 10240, st)
        self.cache.attn_decode(self.table.data_ptr(), self.width, self.len.data_ptr(), n, H, p, 10240, 512,
                               p + 2 * 256, D ** -0.5, self.out.data_ptr(), 4096, self.ws.data_ptr(), self.ws.numel(), st)
        self.wout.gemv(self.out.data_ptr(), n, self.y.data_ptr(), st)

    def read(self, lens):
        k = torch.zeros(int(sum(lens)), KV, D, dtype=torch.bfloat16, device="cuda")
        v = torch.zeros_like(k)
        start, zero = i32(np.concatenate([[0], np.cumsum(lens)])), i32([0] * self.n)
        self.cache.read(self.table.data_ptr(), self.width, zero.data_ptr(), start.data_ptr(), self.n, k.shape[0],
                        k.data_ptr(), KV * D, v.data_ptr(), KV * D)
        torch.cuda.synchronize()
        return list(zip(k.split(list(lens)), v.split(list(lens))))


def prefilled(qcache, synth, lens, a):
    """A context with prompts of these lengths and their projections' K/V."""
    n, pages = len(lens), 16
    q = qcache.QCache(n_attn_layers=1, n_gdn_layers=1, max_seqs=n, max_pages=pages, max_ctx=512, max_batch=n,
                      max_snapshots=1, device=0)
    q.set_attn_params(0, a["q_norm"], a["k_norm"])
    seqs = []
    for i, length in enumerate(lens):
        s = q.seq_alloc()
        proj = synth.attn_inputs(870 + i, length, 0)["proj"]
        for t in range(0, length, 32):
            c = min(32, length - t)
            q.prefill_begin(s, c)
            q.attn_prefill(0, dev(proj[t:t + c]).data_ptr(), empty_u16(c, 4096).data_ptr())
            q.prefill_end()
        seqs.append(s)
    torch.cuda.synchronize()
    q.check_device()
    return q, seqs, pages


def moved(q, seqs, lens, layer):
    """The context's rows into the 8-bit pool, under the context's page ids."""
    tab = np.zeros((len(lens), layer.width), np.int32)
    ks, vs = [], []
    for i, (s, length) in enumerate(zip(seqs, lens)):
        ids = q.seq_pages(s)
        tab[i, : len(ids)] = ids
        k, v = empty_u16(length, KV, D), empty_u16(length, KV, D)
        q.kv_read(s, 0, 0, length, k.data_ptr(), v.data_ptr())
        ks.append(k)
        vs.append(v)
    layer.table.copy_(torch.from_numpy(tab))
    k, v = torch.cat(ks), torch.cat(vs)
    start, zero = i32(np.concatenate([[0], np.cumsum(lens)])), i32([0] * len(lens))
    layer.cache.write(layer.table.data_ptr(), layer.width, zero.data_ptr(), start.data_ptr(), len(lens), k.shape[0],
                      k.data_ptr(), KV * D, v.data_ptr(), KV * D)
    torch.cuda.synchronize()
    return tab


def test_layer_beside_the_bf16_context(qcache, synth, oracle):
    lens = [70, 33, 1, 63]
    n = len(lens)
    a = synth.attn_inputs(860, 1, 0)
    q, seqs, pages = prefilled(qcache, synth, lens, a)
    layer = Layer(qcache, synth, oracle, n, pages, 4, a["q_norm"], a["k_norm"])
    tab = moved(q, seqs, lens, layer)
    at = list(lens)
    for step in range(20):
        layer.x.copy_(torch.from_numpy(synth.gemv_inputs(880 + step, n, HID).view(np.int16)))
        layer.pos.copy_(torch.tensor(at, dtype=torch.int32))
        layer.len.copy_(torch.tensor([p + 1 for p in at], dtype=torch.int32))
        layer.project()
        out_ctx = empty_u16(n, 4096)
        q.decode_begin(seqs)
        q.attn_decode(0, layer.proj.data_ptr(), out_ctx.data_ptr())
        q.decode_end()
        for i, s in enumerate(seqs):
            ids = q.seq_pages(s)
            tab[i, : len(ids)] = ids
        layer.table.copy_(torch.from_numpy(tab))
        raw = layer.proj.clone()
        layer.attend()
        q.check_device()
        qcache.kv8_check()

        rows = bf(layer.proj)
        qr = rows[:, :8192].unflatten(1, (H, 512))
        # gate and v untouched; the rotated k is the one that the context appended, up to
        # the two roundings to bf16 (half a step each) and the context's f32 angles
        assert torch.equal(layer.proj[:, 9216:], raw[:, 9216:])
        assert torch.equal(layer.proj[:, :8192].unflatten(1, (H, 512))[:, :, 256:], raw[:, :8192].unflatten(1, (H, 512))[:, :, 256:])
        for i, s in enumerate(seqs):
            k, v = empty_u16(1, KV, D), empty_u16(1, KV, D)
            q.kv_read(s, 0, at[i], 1, k.data_ptr(), v.data_ptr())
            torch.cuda.synchronize()
            mine, theirs = rows[i, 8192:9216].double(), bf(k).flatten().double()
            assert bool(((mine - theirs).abs() <= 2 * 2.0 ** -8 * theirs.abs() + 1e-4 * theirs.abs().max()).all())
        now = [p + 1 for p in at]
        kvs = layer.read(now)
        check_attention(bf(layer.out).unflatten(1, (H, D)), qr[:, :, :256], qr[:, :, 256:], kvs, D ** -0.5)
        assert_gemv_close(host_u16(layer.y), oracle.bfp8_gemv(layer.packed_out, OUT, 4096, host_u16(layer.out))[1], synth)
        for i, (k, v) in enumerate(kvs):
            g = lambda t: t.double().transpose(0, 1).repeat_interleave(4, 0)  # noqa: E731
            uk, uv = g(k).abs().amax((1, 2)), g(v).abs().amax((1, 2))
            qi = qr[i, :, :256].double()
            d = D ** -0.5 * qi.abs().sum(-1) * uk * 2 / 127
            p = torch.softmax((qi[:, None] @ g(k).transpose(1, 2)).squeeze(1) * D ** -0.5, -1)
            mag = (p[:, None] @ g(v).abs()).squeeze(1)
            bound = torch.expm1(2 * d)[:, None] * mag + (uv * 2 / 127)[:, None]
            mine, theirs = bf(layer.out)[i].unflatten(0, (H, D)).double(), bf(out_ctx)[i].unflatten(0, (H, D)).double()
            tol = bound + 2.0 ** -8 * (mine.abs() + theirs.abs()) + 2e-5
            assert bool(((mine - theirs).abs() <= tol).all())
        at = now
    q.close()


def test_captured_layer_step_replays(qcache, synth, oracle):
    """One captured step replayed 30 times, positions advancing on the device,
    gives the bits of the same steps called one by one."""
    n, steps = 3, 30
    a = synth.attn_inputs(861, 1, 0)
    ids = np.random.default_rng(4).permutation(12).reshape(n, 4).astype(np.int32)
    layers = [Layer(qcache, synth, oracle, n, 12, 4, a["q_norm"], a["k_norm"]) for _ in range(2)]
    torch.cuda.synchronize()
    for layer in layers:
        layer.table.copy_(torch.from_numpy(ids))
        layer.pos.copy_(torch.tensor([0, 50, 9], dtype=torch.int32))
        layer.len.copy_(layer.pos + 1)
    xs = [synth.gemv_inputs(920 + s, n, HID).view(np.int16) for s in range(steps)]
    # positions before the start were never written: zero bytes in both pools, the same finite values
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        st = torch.cuda.current_stream().cuda_stream
        layers[1].project(st)
        layers[1].attend(st)
        layers[1].pos.add_(1)
        layers[1].len.add_(1)
    for s in range(steps):
        for layer in layers:
            layer.x.copy_(torch.from_numpy(xs[s]))
        torch.cuda.synchronize()
        layers[0].project()
        layers[0].attend()
        layers[0].pos.add_(1)
        layers[0].len.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(layers[0].out, layers[1].out) and torch.equal(layers[0].y, layers[1].y)
        assert torch.equal(layers[0].pool, layers[1].pool)
    qcache.kv8_check()
