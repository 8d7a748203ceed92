"""One attention layer of a streaming speech encoder, trained and served.

    python voice-detect.cpp_amd/examples/streaming_attention.py

Three ragged recordings packed one after the other go through a causal layer
with a learned position bias (vdk_rel_bias_expand, vdk_relpos_attention); the
bias's bucket table takes a few gradient steps towards a target
(vdk_relpos_attention_backward, vdk_rel_bias_reduce).  Then the same recordings
are served live: every frame's key and value enters a paged 8-bit cache
(vdk_kv_cache_write) and its query attends over it (vdk_paged_attention), which
gives what the packed call gave, up to the cache's rounding.
"""
import ctypes as C
import math
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from vdamd import lib

LENGTHS, HEADS, KV, DIM, RADIUS, BUCKETS, FAR, CAP, PAGE = [150, 61, 97], 8, 4, 64, 64, 16, 64, 30.0, 32
RATE = 1.0   # of the mean gradient of a frame


def half(rng, *shape):
    return rng.standard_normal(shape).astype(np.float16)


class Layer:
    """Device buffers and descriptors of one packed layout; a step is forward and backward."""

    def __init__(self, q, k, v):
        n = q.shape[0]
        self.L, self.n, self.at = lib.lib(), n, np.concatenate([[0], np.cumsum(LENGTHS)]).tolist()
        self.plan = lib.AttnPlan(self.at, self.at, HEADS, KV, DIM, causal=True)
        self.buf = {"q": lib.DeviceBuffer.from_array(q), "k": lib.DeviceBuffer.from_array(k),
                    "v": lib.DeviceBuffer.from_array(v)}
        size = self.L.vdk_relpos_attention_backward_workspace_size(self.plan.ptr, RADIUS)
        for name, nbytes in (("o", n * HEADS * DIM * 2), ("o32", n * HEADS * DIM * 4), ("lse", HEADS * n * 4),
                             ("do", n * HEADS * DIM * 2), ("dq", n * HEADS * DIM * 2), ("dk", n * KV * DIM * 2),
                             ("dv", n * KV * DIM * 2), ("table", BUCKETS * HEADS * 4), ("dtable", BUCKETS * HEADS * 4),
                             ("dist", HEADS * (2 * RADIUS + 1) * 4), ("ddist", HEADS * (2 * RADIUS + 1) * 4),
                             ("work", size)):
            self.buf[name] = lib.DeviceBuffer(nbytes)
        b = {name: x.ptr for name, x in self.buf.items()}
        a = self.attn = lib.RelposAttn()
        a.dtype, a.scale, a.cap = lib.F16, 1 / math.sqrt(DIM), CAP
        for x, h in (("q", HEADS), ("k", KV), ("v", KV), ("o", HEADS)):
            setattr(a, x, b[x])
            setattr(a, x + "_tok", h * DIM)
            setattr(a, x + "_head", DIM)
        a.dist_bias, a.bias_radius, a.o_f32, a.lse = b["dist"], RADIUS, b["o32"], b["lse"]
        g = self.grad = lib.RelposAttnGrad()
        for x, y, h in (("d_o", "do", HEADS), ("dq", "dq", HEADS), ("dk", "dk", KV), ("dv", "dv", KV)):
            setattr(g, x, b[y])
            setattr(g, y + "_tok", h * DIM)
            setattr(g, y + "_head", DIM)
        g.d_dist_bias, g.work, g.work_bytes = b["ddist"], b["work"], size

    def forward(self, table):
        b = self.buf
        b["table"].copy_from(table.astype(np.float32))
        lib.check(self.L.vdk_rel_bias_expand(b["table"].ptr, BUCKETS, HEADS, 0, FAR, RADIUS, b["dist"].ptr, None))
        lib.check(self.L.vdk_relpos_attention(self.plan.ptr, self.attn, None))
        return b["o"].to_array(np.float16, (self.n, HEADS, DIM)).astype(np.float32)

    def backward(self, do):
        b = self.buf
        b["do"].copy_from(do.astype(np.float16))
        lib.check(self.L.vdk_relpos_attention_backward(self.plan.ptr, self.attn, self.grad, None))
        lib.check(self.L.vdk_rel_bias_reduce(b["ddist"].ptr, BUCKETS, HEADS, 0, FAR, RADIUS, b["dtable"].ptr, None))
        return b["dtable"].to_array(np.float32, (BUCKETS, HEADS))


class Streams:
    """The recordings' cache, and one frame of each a step."""

    def __init__(self, dist):
        self.L, self.n = lib.lib(), len(LENGTHS)
        per = max(-(-x // PAGE) for x in LENGTHS)
        pages = per * self.n
        order = np.random.default_rng(3).permutation(pages).astype(np.int32).reshape(self.n, per)
        self.order, rows = order, pages * KV * PAGE
        self.buf = {"k": lib.DeviceBuffer(rows * DIM), "v": lib.DeviceBuffer(rows * DIM), "ks": lib.DeviceBuffer(rows * 4),
                    "vs": lib.DeviceBuffer(rows * 4), "table": lib.DeviceBuffer.from_array(order),
                    "status": lib.DeviceBuffer.from_array(np.zeros(1, np.int32)), "slots": lib.DeviceBuffer(8 * self.n),
                    "lens": lib.DeviceBuffer(4 * self.n), "newk": lib.DeviceBuffer(self.n * KV * DIM * 2),
                    "newv": lib.DeviceBuffer(self.n * KV * DIM * 2), "q": lib.DeviceBuffer(self.n * HEADS * DIM * 2),
                    "o": lib.DeviceBuffer(self.n * HEADS * DIM * 2)}
        b = {name: x.ptr for name, x in self.buf.items()}
        c = self.cache = lib.KvCache()
        c.dtype, c.format, c.n_pages, c.page_size, c.n_kv_heads, c.head_dim = lib.F16, lib.KV_E4M3, pages, PAGE, KV, DIM
        c.k, c.v, c.k_scale, c.v_scale = b["k"], b["v"], b["ks"], b["vs"]
        a = self.attn = lib.PagedAttn()
        a.n_seqs, a.n_q_heads, a.max_pages, a.max_len = self.n, HEADS, per, max(LENGTHS)
        a.q, a.o, a.q_seq, a.o_seq, a.q_head, a.o_head = b["q"], b["o"], HEADS * DIM, HEADS * DIM, DIM, DIM
        a.block_table, a.seq_lens, a.status = b["table"], b["lens"], b["status"]
        a.scale, a.cap, a.dist_bias, a.bias_radius = 1 / math.sqrt(DIM), CAP, dist.ptr, RADIUS
        size = self.L.vdk_paged_attention_workspace_size(c, a)
        self.work = lib.DeviceBuffer(size)
        a.work, a.work_bytes = self.work.ptr, size

    def step(self, t, q, k, v):
        """Frame t of every stream (those that have ended keep their last length); the outputs."""
        b = self.buf
        live = np.array([t < x for x in LENGTHS])
        slots = np.where(live, self.order[:, min(t, max(LENGTHS) - 1) // PAGE].astype(np.int64) * PAGE + t % PAGE, -1)
        for name, x in (("slots", slots.view(np.uint8)), ("newk", k), ("newv", v), ("q", q),
                        ("lens", np.minimum(t + 1, LENGTHS).astype(np.int32))):
            b[name].copy_from(x)
        lib.check(self.L.vdk_kv_cache_write(self.cache, b["slots"].ptr, self.n, b["newk"].ptr, KV * DIM, DIM,
                                            b["newv"].ptr, KV * DIM, DIM, b["status"].ptr, None))
        lib.check(self.L.vdk_paged_attention(self.cache, self.attn, None))
        return b["o"].to_array(np.float16, (self.n, HEADS, DIM)).astype(np.float32)


def main():
    rng = np.random.default_rng(1)
    n = sum(LENGTHS)
    q, k, v = half(rng, n, HEADS, DIM), half(rng, n, KV, DIM), half(rng, n, KV, DIM)
    layer = Layer(q, k, v)

    # the target: the same layer under another bias; the loss is half the squared distance, a frame and head
    target = layer.forward(rng.standard_normal((BUCKETS, HEADS)))
    table, losses = np.zeros((BUCKETS, HEADS), np.float32), []
    for _ in range(30):
        o = layer.forward(table)
        losses.append(float(0.5 * ((o - target) ** 2).sum() / n))
        table -= RATE * layer.backward(o - target) / n
    print(f"training the position bias: loss {losses[0]:.4f} -> {losses[-1]:.4f} in {len(losses)} steps")

    packed = layer.forward(table)
    streams = Streams(layer.buf["dist"])
    worst = square = 0.0
    for t in range(max(LENGTHS)):
        rows = [at + min(t, x - 1) for at, x in zip(layer.at, LENGTHS)]
        out = streams.step(t, q[rows], k[rows], v[rows])
        for i, x in enumerate(LENGTHS):
            if t < x:
                d = out[i] - packed[rows[i]]
                worst, square = max(worst, float(np.abs(d).max())), square + float((d ** 2).sum())
    rms = math.sqrt(square / packed.size)
    status = int(streams.buf["status"].to_array(np.int32, (1,))[0])
    print(f"served frame by frame over an 8-bit cache: rms difference {rms:.4f}, largest {worst:.4f}, status {status}")
    return losses, rms, float(packed.std()), status


if __name__ == "__main__":
    main()
