"""The paged operators together, as a serving loop uses them: decode steps of a small model for sequences of their own lengths -- norm, one packed q/k/v
product, append with norms and rotation, attention over the pages, output product, logits, sampling -- eagerly and as a replayed graph, against the same in 64 bits on the
dequantized weights."""
import numpy as np
import pytest

from oracle import oracle as orc
from test_gpu_decode_ops import np_rmsnorm, np_rope
from test_gpu_sample import reference
from torchlette_b200 import backend as tb

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV, DIM, VOCAB, PAGE, EPS = 256, 4, 2, 64, 1000, 16, 1e-6


class Model:
    def __init__(self, be, rng):
        self.be = be

        def packed(n, k):
            w = (rng.standard_normal((n, k)) / np.sqrt(k)).astype(np.float32)
            p, s = be.quantizeLinearWeight(w, 64)
            return be.createQuantizedWeight(p, s, n, k, tb.resolveWeightFormat("int8-64")), orc.dequantize_to_f32(p, s, k, 64).astype(np.float64)

        self.qkv, self.qkv_r = packed((HEADS + 2 * KV) * DIM, HIDDEN)
        self.o, self.o_r = packed(HIDDEN, HEADS * DIM)
        self.head, self.head_r = packed(VOCAB, HIDDEN)
        self.norms = {n: rng.uniform(0.5, 1.5, w).astype(np.float32) for n, w in (("in", HIDDEN), ("q", DIM), ("k", DIM), ("out", HIDDEN))}
        self.t = {n: be.ops.tensorFromArray(w, list(w.shape), "f32") for n, w in self.norms.items()}
        angle = np.arange(200)[:, None] / 1e4 ** (np.arange(DIM // 2)[None, :] / (DIM // 2))
        self.cos, self.sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
        self.t["cos"], self.t["sin"] = (be.ops.tensorFromArray(a, list(a.shape), "f32") for a in (self.cos, self.sin))
        self.embedding = rng.standard_normal((VOCAB, HIDDEN)).astype(np.float32)

    def step(self, x, cache, positions, uniforms, temperature, topK, topP, hold):
        ops, be = self.be.ops, self.be
        h0 = ops.rmsnorm(x, self.t["in"], EPS)
        qkv = be.linear(h0, self.qkv)
        q = ops.pagedAppend(cache, positions, qkv, None, None, self.t["cos"], self.t["sin"], qNorm=self.t["q"], kNorm=self.t["k"], eps=EPS, out=hold["q"])
        a = ops.pagedAttention(cache, positions, q, DIM ** -0.5, out=hold["a"])
        o = be.linear(a, self.o)
        h1 = ops.add(x, o)
        h2 = ops.rmsnorm(h1, self.t["out"], EPS)
        ops.matmul(h2, ops.transpose(self.head), {"outBuffer": hold["logits"], "outputDtype": "f32"})
        ops.sample(hold["logits"], uniforms, temperature=temperature, topK=topK, topP=topP, out=hold["tokens"])
        for t in (h0, qkv, o, h1, h2):
            t.destroy()

    def reference(self, x, past, pos):
        """logits of one sequence, whose keys and values are appended to `past`"""
        qkv = np_rmsnorm(x, self.norms["in"], EPS) @ self.qkv_r.T
        q, k, v = np.split(qkv.reshape(-1, DIM), [HEADS, HEADS + KV])
        q, k = (np_rope(np_rmsnorm(a, self.norms[n], EPS)[:, None], self.cos[pos:pos + 1], self.sin[pos:pos + 1])[:, 0] for a, n in ((q, "q"), (k, "k")))
        past.append((k, v))
        keys, values = (np.repeat(np.stack([p[i] for p in past]), HEADS // KV, 1) for i in (0, 1))
        s = np.einsum("hd,jhd->hj", q, keys) * DIM ** -0.5
        w = np.exp(s - s.max(1, keepdims=True))
        a = np.einsum("hj,jhd->hd", w / w.sum(1, keepdims=True), values).reshape(-1)
        return np_rmsnorm(x + a @ self.o_r.T, self.norms["out"], EPS) @ self.head_r.T


@pytest.mark.parametrize("replayed", [False, True])
def test_decode_steps_of_sequences_of_their_own_lengths(backend, replayed):
    be, seqs, steps = backend, 3, 36
    rng = np.random.default_rng(31)
    m = Model(be, rng)
    ops = be.ops
    start = [0, 17, 5]  # how far each is when the loop begins; the third is not there for some steps
    pages, width = 20, 5
    table = rng.permutation(pages)[:seqs * width].reshape(seqs, width).astype(np.int32)
    up = lambda a, dtype: ops.tensorFromArray(a, list(a.shape), dtype)  # noqa: E731
    kp, vp = (up(np.full((pages, KV, PAGE, DIM), np.nan, np.float32), "f32") for _ in range(2))
    cache = be.createPagedCache(kp, vp, up(table, "i32"))
    dev = {"x": up(np.zeros((seqs, HIDDEN), np.float32), "f32"), "pos": up(np.zeros(seqs, np.int32), "i32"), "u": up(np.zeros(seqs, np.float32), "f32"),
           "t": up(np.array([0.8, 0.0, 1.1], np.float32), "f32"), "k": up(np.array([40, 0, 0], np.int32), "i32"), "p": up(np.array([0.9, 1.0, 0.95], np.float32), "f32")}
    hold = {"q": ops.empty([seqs, HEADS, DIM], "f32"), "a": ops.empty([seqs, HEADS * DIM], "f32"), "logits": ops.empty([seqs, VOCAB], "f32"),
            "tokens": ops.empty([seqs], "i32")}
    past = [[], [], []]
    # what is there before the loop: prompts, appended in one call of all their tokens
    prompt = [(s, p) for s in range(seqs) for p in range(start[s])]
    kv = [rng.standard_normal((len(prompt), KV, DIM)).astype(np.float32) for _ in range(2)]
    for (s, _), k, v in zip(prompt, *kv):
        past[s].append((k.astype(np.float64), v.astype(np.float64)))
    ops.pagedAppend(cache, up(np.array([p for _, p in prompt], np.int32), "i32"), None, up(kv[0], "f32"), up(kv[1], "f32"),
                    tokenSeq=up(np.array([s for s, _ in prompt], np.int32), "i32"))
    run = lambda: m.step(dev["x"], cache, dev["pos"], dev["u"], dev["t"], dev["k"], dev["p"], hold)  # noqa: E731
    be._upload(dev["pos"].buffer, np.full(seqs, -1, np.int32))
    run()  # scratch, and the blocks that a capture may take from the pool
    be.sync()
    graph = None
    kept = []
    if replayed:
        # nothing can be allocated while a stream is captured: the captured step gets the temporaries of a step before it, which stay
        class Ops(tb.CudaOps):
            def empty(self, shape, dtype="f32"):
                if graph_of is None:
                    kept.append(tb.CudaOps.empty(self, shape, dtype))
                    return tb.CudaTensor(be, shape, dtype, kept[-1].buffer, kept[-1].nbytes, ownsBuffer=False)
                t = kept[next(graph_of)]
                assert t.shape == list(shape) and t.dtype == dtype
                return tb.CudaTensor(be, shape, dtype, t.buffer, t.nbytes, ownsBuffer=False)

        graph_of, be.ops = None, Ops(be)
        try:
            run()
            be.sync()
            graph_of = iter(range(len(kept)))
            be.beginCapture()
            run()
            graph = be.endCapture()
        finally:
            be.ops = ops
    token = [1, 2, 3]
    for step in range(steps):
        there = [True, True, step % 7 != 3]
        pos = [len(past[s]) if there[s] else -1 for s in range(seqs)]
        x = m.embedding[token].copy()
        u = rng.uniform(size=seqs).astype(np.float32)
        for n, a in (("x", x), ("pos", np.array(pos, np.int32)), ("u", u)):
            be._upload(dev[n].buffer, a)
        if graph:
            be.replay(graph)
        else:
            run()
        logits, tokens = ops.read(hold["logits"]), ops.read(hold["tokens"])
        for s in range(seqs):
            if not there[s]:
                continue
            ref = m.reference(x[s].astype(np.float64), past[s], pos[s])
            assert np.max(np.abs(logits[s] - ref) / np.maximum(1.0, np.abs(ref))) <= 1e-3
            params = [(0.8, 40, 0.9), (0.0, 0, 1.0), (1.1, 0, 0.95)][s]
            want = reference(logits[s].astype(np.float64), float(u[s]), float(np.float32(params[0])), params[1], float(np.float32(params[2])))
            assert tokens[s] == want
            token[s] = int(tokens[s])
    be.sync()
    if graph:
        be.destroyGraph(graph)
        for t in kept:
            t.destroy()
