"""Attention with a learned position bias, packed clips, masks and capped scores, its
training step, its single-frame form over a paged cache, and that cache's quantised writing.

A case is a dict of plain values.  listed() gives the named cases, draw(rng)
another one of the same ranges, prepare(case, seed) what a program has in hand
before the call, run(state) one pass, work(case) the bytes and operations that
pass cannot do without, exact(case, seed) the same outputs in 64 bits.  With
`own` false run() computes the operators in elementary torch operations, with
`own` true through the framework's entry points.

Kinds of case:
  attend  packed clips of uneven length through one attention layer (vdk_relpos_attention)
  train   the same layer's training step: the bias from its bucket table, the outputs and all
          gradients (vdk_rel_bias_expand, vdk_relpos_attention, vdk_relpos_attention_backward,
          vdk_rel_bias_reduce)
  decode  one new frame of every stream over a paged cache (vdk_paged_attention)
  cache   new frames written to that cache and read back (vdk_kv_cache_write, vdk_kv_cache_read)

For query i and key j of a clip, with r = j - (i + past) their distance:
  x = scale * q_i . k_j,  s = cap * tanh(x / cap) + bias[head][clamp(r, -R, R) + R]
  (s = x + bias without a cap), keys past the query hidden if causal, but for
  the clip's first `prefix` keys; o_i = sum_j softmax_j(s) v_j, lse_i = log sum_j exp(s).
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
E4M3_MAX = 448.0
TINY = 2.0 ** -64   # smallest magnitude a quantised row is scaled by


# ------------------------------------------------------------------ the cases

def _attend(name, docs, lo, hi, heads, kv, dim, dtype, bias=0, cap=0.0, causal=False, prefix=0, past=0):
    return {"name": name, "kind": "attend", "docs": docs, "lo": lo, "hi": hi, "heads": heads, "kv": kv, "dim": dim,
            "dtype": dtype, "bias": bias, "cap": cap, "causal": causal, "prefix": prefix, "past": past}


def _train(name, docs, lo, hi, heads, kv, dim, dtype, bias=0, cap=0.0, causal=False, prefix=0):
    return dict(_attend(name, docs, lo, hi, heads, kv, dim, dtype, bias, cap, causal, prefix), kind="train")


def _decode(name, seqs, lo, hi, heads, kv, dim, dtype, quant, page, bias=0, cap=0.0):
    return {"name": name, "kind": "decode", "docs": seqs, "lo": lo, "hi": hi, "heads": heads, "kv": kv, "dim": dim,
            "dtype": dtype, "quant": quant, "page": page, "bias": bias, "cap": cap}


def _cache(name, tokens, pages, kv, dim, dtype, quant, page):
    return {"name": name, "kind": "cache", "tokens": tokens, "pages": pages, "kv": kv, "dim": dim, "dtype": dtype,
            "quant": quant, "page": page}


def listed():
    return [
        # one 3 s clip in the base analyze model's heads: a single file, bound by latency
        _attend("attend_1x149", 1, 149, 149, 12, 12, 64, "f16", bias=128),
        # a batch of clips as a voice-activity detector cuts them (0.5 to 10 s), packed
        _attend("attend_32xragged", 32, 24, 499, 16, 16, 64, "f16", bias=800),
        # one whole recording of four minutes, every frame seeing every other
        _attend("attend_1x12001", 1, 12001, 12001, 16, 16, 64, "bf16", bias=800),
        # a chunk of a live recording over its history: shared heads, capped scores, causal
        _attend("attend_chunk_8x512", 8, 400, 512, 16, 4, 128, "bf16", cap=30.0, causal=True, past=2048),
        # fine-tuning on a handful of short clips
        _train("train_4xragged", 4, 60, 149, 12, 12, 64, "f16", bias=128),
        # fine-tuning on a batch of 3 to 16 s clips with the learned bias
        _train("train_16xragged", 16, 149, 799, 16, 16, 64, "bf16", bias=800),
        # a causal streaming encoder trained on long recordings, with a prefix that all frames see
        _train("train_causal_2x4096", 2, 3900, 4096, 16, 4, 64, "bf16", bias=128, cap=50.0, causal=True, prefix=100),
        # one live stream, a few seconds in: the smallest call
        _decode("decode_1x500", 1, 500, 500, 12, 12, 64, "f16", False, 16, bias=128),
        # many live streams of up to half a minute over an 8-bit cache
        _decode("decode_64x1500", 64, 200, 1500, 16, 16, 64, "f16", True, 32, bias=800),
        # hour-long recordings (20 ms frames would be 180000 a head; here up to 65000), shared heads
        _decode("decode_12x65000", 12, 9000, 65000, 32, 8, 128, "bf16", True, 64, cap=30.0),
        # the streams' new frames written each step
        _cache("cache_64", 64, 2048, 16, 64, "f16", True, 32),
        # a batch of whole recordings written at once
        _cache("cache_20011", 20011, 1024, 8, 128, "bf16", True, 64),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["attend", "attend", "train", "train", "decode", "decode", "cache"])
        dim = rng.choice([64, 64, 128])
        kv = rng.choice([1, 2, 4, 8, 12, 16])
        heads = kv * rng.choice([1, 1, 2, 4, 8])
        dtype = rng.choice(["f16", "bf16"])
        if heads > 32:
            continue
        bias, cap = rng.choice([0, 128, 800]), rng.choice([0.0, 0.0, 20.0, 50.0])
        if kind == "cache":
            page = rng.choice([16, 32, 64, 128])
            n = _log_int(rng, 1, 20000)
            c = _cache("", n, -(-n // page) + rng.randint(1, 500), kv, dim, dtype, rng.random() < 0.7, page)
        elif kind == "decode":
            hi = _log_int(rng, 1, 65000)
            c = _decode("", _log_int(rng, 1, 128), max(1, int(hi * rng.random())), hi, heads, kv, dim, dtype,
                        rng.random() < 0.6, rng.choice([16, 32, 64, 128]), bias, cap)
        else:
            # (a clip of one frame has no gradient but its values', so training draws longer ones among them)
            hi = _log_int(rng, 1, 8192) if kind == "attend" else _log_int(rng, 8, 4096)
            causal = rng.random() < 0.5
            c = _attend("", _log_int(rng, 1, 64), max(1, int(hi * rng.random())), hi, heads, kv, dim, dtype, bias,
                        cap, causal, rng.choice([0, 0, _log_int(rng, 1, hi)]) if causal else 0,
                        _log_int(rng, 1, 2000) if kind == "attend" and causal and rng.random() < 0.4 else 0)
            c["kind"] = kind
        del c["name"]
        if _within(c):
            return c


def _within(c):
    """Whether a drawn case costs no more than the largest listed one of its kind, in memory of the plain form too."""
    same = [d for d in listed() if d["kind"] == c["kind"]]
    w, most = work(c), [work(d) for d in same]
    if w["bytes"] > max(m["bytes"] for m in most) or w["flops"] > max(m["flops"] for m in most):
        return False
    if c["kind"] in ("attend", "train"):
        return _pairs(c) <= max(_pairs(d) for d in same)
    return c["kind"] == "cache" or c["docs"] * c["hi"] * c["kv"] * c["dim"] <= 12 * 65000 * 8 * 128


def _pairs(c):
    return c["docs"] * c["heads"] * c["hi"] * (c["hi"] + c.get("past", 0))


def _lengths(c):
    """The clips' lengths, the longest always among them."""
    r = random.Random(c["docs"] * 1000003 + c["lo"] * 1009 + c["hi"])
    n = [r.randint(c["lo"], c["hi"]) for _ in range(c["docs"])]
    n[r.randrange(c["docs"])] = c["hi"]
    return n


def _buckets(c):
    """(buckets of the bias table, distance from which all share the last one)."""
    return {128: (32, 128), 800: (320, 800)}[c["bias"]]


# -------------------------------------------------------------------- prepare

def _normal(g, shape, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def _offsets(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at


def _quantise(x):
    """Rows of x as e4m3 codes and the scale of each: code * scale is the value.  x * E4M3_MAX is exact
    (x has 11 bits at most) and the quotient's one rounding keeps a tie between two codes a tie."""
    x = x.float()
    most = x.abs().amax(-1, keepdim=True).clamp_min(TINY)
    return (x * E4M3_MAX / most).to(torch.float8_e4m3fn), (most / E4M3_MAX).squeeze(-1)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    st = {"case": case}
    t, D, kv = TYPES[case["dtype"]], case["dim"], case["kv"]
    if case["kind"] in ("attend", "train"):
        H, n = case["heads"], _lengths(case)
        st["q_at"], st["kv_at"] = _offsets(n), _offsets([x + case["past"] for x in n])
        nq, nk = st["q_at"][-1], st["kv_at"][-1]
        st["q_off"] = torch.tensor(st["q_at"], device=DEV)
        st["kv_off"] = torch.tensor(st["kv_at"], device=DEV)
        st["prefix_of"] = [min(case["prefix"], x + case["past"]) for x in n]
        st["prefix"] = torch.tensor(st["prefix_of"], device=DEV)
        # queries, keys and values as one projection's output holds them
        if case["past"]:
            st["q"] = _normal(g, (nq, H, D), 1.2, t)
            st["k"], st["v"] = _normal(g, (nk, 2 * kv, D), 1.0, t).split([kv, kv], 1)
        else:
            st["q"], st["k"], st["v"] = _normal(g, (nq, H + 2 * kv, D), 1.1, t).split([H, kv, kv], 1)
        if case["bias"]:
            nb, _ = _buckets(case)
            st["table"] = _normal(g, (nb, H), 1.0)
            st["dist"] = _expand(case, st["table"])
        if case["kind"] == "train":
            st["do"] = _normal(g, (nq, H, D), 0.05, t)
    elif case["kind"] == "decode":
        H, page = case["heads"], case["page"]
        n = _lengths(case)
        per = [-(-x // page) for x in n]
        pages = sum(per) + 3
        order = torch.randperm(pages, generator=g, device=DEV)   # as streams that come and go leave them
        table = torch.zeros(len(n), max(per), dtype=torch.int32, device=DEV)
        at = 0
        for i, p in enumerate(per):
            table[i, :p] = order[at:at + p]
            at += p
        st["pages"], st["lens"] = table, torch.tensor(n, dtype=torch.int32, device=DEV)
        st["q"] = _normal(g, (len(n), H, D), 1.2, t)
        for x in ("k", "v"):
            new = _normal(g, (pages, kv, page, D), 1.0, t)
            st[x + "_cache"], st[x + "_scale"] = _quantise(new) if case["quant"] else (new, None)
        if case["bias"]:
            nb, _ = _buckets(case)
            st["dist"] = _expand(case, _normal(g, (nb, H), 1.0))
    else:
        n, pages, page = case["tokens"], case["pages"], case["page"]
        st["slots"] = torch.randperm(pages * page, generator=g, device=DEV)[:n].contiguous()
        st["k"], st["v"] = _normal(g, (n, 2 * kv, D), 1.0, t).split([kv, kv], 1)
        for x in ("k", "v"):
            shape = (pages, kv, page, D)
            st[x + "_cache"] = torch.zeros(shape, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) \
                if case["quant"] else torch.zeros(shape, dtype=t, device=DEV)
            st[x + "_scale"] = torch.zeros(shape[:3], device=DEV) if case["quant"] else None
    if own:
        _bind(st)
    torch.cuda.synchronize()
    return st


# -------------------------------------------------- the framework's own calls

def _ptr(x):
    return None if x is None else x.data_ptr()


def _bind(st):
    """The descriptors, the plan of the clips' layout, the outputs and the workspace a program keeps."""
    import os
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    sys.path.insert(0, os.path.join(root, "voice-detect.cpp_amd"))
    from vdamd import lib
    L, c = lib.lib(), st["case"]
    t, D, kv = TYPES[c["dtype"]], c["dim"], c["kv"]
    code = lib.BF16 if c["dtype"] == "bf16" else lib.F16
    st["lib"], st["L"] = lib, L
    st["stream"] = torch.cuda.current_stream().cuda_stream
    if c["kind"] in ("attend", "train"):
        H, nq = c["heads"], st["q"].shape[0]
        st["plan"] = lib.AttnPlan(st["q_at"], st["kv_at"], H, kv, D, causal=c["causal"], prefix=st["prefix_of"])
        a = lib.RelposAttn()
        a.dtype, a.scale, a.cap = code, 1 / math.sqrt(D), c["cap"]
        for x in ("q", "k", "v"):
            setattr(a, x, st[x].data_ptr())
            setattr(a, x + "_tok", st[x].stride(0))
            setattr(a, x + "_head", st[x].stride(1))
        if c["bias"]:
            if c["kind"] == "train":
                st["dist"] = torch.empty(H, 2 * c["bias"] + 1, device=DEV)
            a.dist_bias, a.bias_radius = st["dist"].data_ptr(), c["bias"]
        st["o"], st["lse"] = torch.empty(nq, H, D, dtype=t, device=DEV), torch.empty(H, nq, device=DEV)
        a.o, a.o_tok, a.o_head, a.lse = st["o"].data_ptr(), H * D, D, st["lse"].data_ptr()
        if c["kind"] == "train":
            st["o32"] = torch.empty(nq, H, D, device=DEV)
            a.o_f32 = st["o32"].data_ptr()
            b = lib.RelposAttnGrad()
            b.d_o, b.do_tok, b.do_head = st["do"].data_ptr(), H * D, D
            st["dq"] = torch.empty(nq, H, D, dtype=t, device=DEV)
            st["dk"], st["dv"] = (torch.empty(nq, kv, D, dtype=t, device=DEV) for _ in range(2))
            b.dq, b.dq_tok, b.dq_head = st["dq"].data_ptr(), H * D, D
            b.dk, b.dk_tok, b.dk_head = st["dk"].data_ptr(), kv * D, D
            b.dv, b.dv_tok, b.dv_head = st["dv"].data_ptr(), kv * D, D
            if c["bias"]:
                st["ddist"] = torch.empty(H, 2 * c["bias"] + 1, device=DEV)
                st["dtable"] = torch.empty_like(st["table"])
                b.d_dist_bias = st["ddist"].data_ptr()
            n = L.vdk_relpos_attention_backward_workspace_size(st["plan"].ptr, c["bias"])
            st["work"] = torch.empty(n, dtype=torch.uint8, device=DEV)
            b.work, b.work_bytes = st["work"].data_ptr(), n
            st["grad"] = b
        st["attn"] = a
        return
    st["status"] = torch.zeros(1, dtype=torch.int32, device=DEV)
    d = lib.KvCache()
    d.dtype, d.format = code, lib.KV_E4M3 if c["quant"] else lib.KV_16
    d.n_pages, d.page_size, d.n_kv_heads, d.head_dim = st["k_cache"].shape[0], c["page"], kv, D
    d.k, d.v, d.k_scale, d.v_scale = (_ptr(st[x]) for x in ("k_cache", "v_cache", "k_scale", "v_scale"))
    st["kvc"] = d
    if c["kind"] == "decode":
        H, n = c["heads"], c["docs"]
        a = lib.PagedAttn()
        a.n_seqs, a.n_q_heads, a.max_pages, a.max_len = n, H, st["pages"].shape[1], c["hi"]
        a.q, a.q_seq, a.q_head = st["q"].data_ptr(), H * D, D
        a.block_table, a.seq_lens = st["pages"].data_ptr(), st["lens"].data_ptr()
        a.scale, a.cap = 1 / math.sqrt(D), c["cap"]
        if c["bias"]:
            a.dist_bias, a.bias_radius = st["dist"].data_ptr(), c["bias"]
        st["o"], st["lse"] = torch.empty(n, H, D, dtype=t, device=DEV), torch.empty(n, H, device=DEV)
        a.o, a.o_seq, a.o_head, a.lse = st["o"].data_ptr(), H * D, D, st["lse"].data_ptr()
        size = L.vdk_paged_attention_workspace_size(d, a)
        st["work"] = torch.empty(max(size, 1), dtype=torch.uint8, device=DEV)
        a.work, a.work_bytes, a.status = st["work"].data_ptr(), size, st["status"].data_ptr()
        st["paged"] = a
    else:
        st["k_back"], st["v_back"] = (torch.empty(c["tokens"], kv, D, dtype=t, device=DEV) for _ in range(2))


def _own_run(st):
    lib, L, c, s = st["lib"], st["L"], st["case"], st["stream"]
    if c["kind"] == "attend":
        lib.check(L.vdk_relpos_attention(st["plan"].ptr, st["attn"], s))
        return {"o": st["o"], "lse": st["lse"]}
    if c["kind"] == "train":
        out = {"o": st["o"], "lse": st["lse"], "dq": st["dq"], "dk": st["dk"], "dv": st["dv"]}
        if c["bias"]:
            nb, far = _buckets(c)
            lib.check(L.vdk_rel_bias_expand(st["table"].data_ptr(), nb, c["heads"], 1, far, c["bias"],
                                            st["dist"].data_ptr(), s))
        lib.check(L.vdk_relpos_attention(st["plan"].ptr, st["attn"], s))
        lib.check(L.vdk_relpos_attention_backward(st["plan"].ptr, st["attn"], st["grad"], s))
        if c["bias"]:
            lib.check(L.vdk_rel_bias_reduce(st["ddist"].data_ptr(), nb, c["heads"], 1, far, c["bias"],
                                            st["dtable"].data_ptr(), s))
            out["dtable"] = st["dtable"]
        return out
    if c["kind"] == "decode":
        lib.check(L.vdk_paged_attention(st["kvc"], st["paged"], s))
        return {"o": st["o"], "lse": st["lse"]}
    n, kv, D = c["tokens"], c["kv"], c["dim"]
    k, v = st["k"], st["v"]
    lib.check(L.vdk_kv_cache_write(st["kvc"], st["slots"].data_ptr(), n, k.data_ptr(), k.stride(0), k.stride(1),
                                   v.data_ptr(), v.stride(0), v.stride(1), st["status"].data_ptr(), s))
    lib.check(L.vdk_kv_cache_read(st["kvc"], st["slots"].data_ptr(), n, st["k_back"].data_ptr(), kv * D, D,
                                  st["v_back"].data_ptr(), kv * D, D, st["status"].data_ptr(), s))
    return _cache_outputs(st)


def _cache_outputs(st):
    out = {"k": st["k_back"], "v": st["v_back"]}
    if st["case"]["quant"]:
        out["k_scale"], out["v_scale"] = st["k_scale"], st["v_scale"]
    else:
        out["k_cache"], out["v_cache"] = st["k_cache"], st["v_cache"]
    return out


# ------------------------------------------------------------ the plain forms

def _bucket(rel, buckets, far):
    """The bucket of each distance: half of them for keys after the query; in each half the
    first half for one distance each, the others for ranges that widen with its logarithm."""
    half = buckets // 2
    near = half // 2
    d = rel.abs().double()
    wide = near + torch.floor(torch.log(d.clamp_min(1) / near) / math.log(far / near) * (half - near) + 1e-9)
    b = torch.where(d < near, d, wide.clamp_max(half - 1)).long()
    return b + half * (rel > 0)


def _expand(case, table):
    """The bias of each head [heads][2 R + 1] at distances -R .. R."""
    R = case["bias"]
    nb, far = _buckets(case)
    return table[_bucket(torch.arange(-R, R + 1, device=DEV), nb, far)].t().contiguous()


def _padded(x, off, longest):
    """Packed rows [n][h][d] as [clip][h][longest][d] in 32 bits, zero past a clip's end."""
    i = off[:-1, None] + torch.arange(longest, device=DEV)
    ok = (i < off[1:, None])[..., None, None]
    y = torch.where(ok, x[i.clamp_max(x.shape[0] - 1)].float(), torch.zeros((), device=DEV))
    return y.permute(0, 2, 1, 3).contiguous()


def _packed(x, off):
    """The clips' rows of [clip][h][longest][d], one after the other."""
    ok = torch.arange(x.shape[2], device=DEV) < (off[1:] - off[:-1])[:, None]
    return x.transpose(1, 2)[ok]


def _softmax(s):
    """(probabilities, log of the sum) over the last axis; a row that sees nothing gives zeros and -inf."""
    m = s.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total > 0, total, torch.ones_like(total))
    return p, (m + torch.log(total)).squeeze(-1)


def _plain_attend(st):
    c = st["case"]
    H, kv, D, R = c["heads"], c["kv"], c["dim"], c["bias"]
    n, Lq, Lk = c["docs"], c["hi"], c["hi"] + c["past"]
    nq, nk = (st[x][1:] - st[x][:-1] for x in ("q_off", "kv_off"))
    q = _padded(st["q"], st["q_off"], Lq).view(n * kv, -1, D)     # a shared head's queries one after the other
    k = _padded(st["k"], st["kv_off"], Lk).view(n * kv, Lk, D)
    v = _padded(st["v"], st["kv_off"], Lk).view(n * kv, Lk, D)
    scale = 1 / math.sqrt(D)
    s = torch.bmm(q, k.transpose(1, 2).contiguous()).view(n, H, Lq, Lk)
    s *= scale
    t = None
    if c["cap"]:
        t = torch.tanh(s / c["cap"])
        s = t * c["cap"]
    i, j = torch.arange(Lq, device=DEV)[:, None], torch.arange(Lk, device=DEV)[None, :]
    rel = j - (i + c["past"])
    if R:
        bias = _expand(c, st["table"]) if c["kind"] == "train" else st["dist"]
        s += bias[:, rel.clamp(-R, R) + R]
    seen = (i < nq[:, None, None]) & (j < nk[:, None, None])
    if c["causal"]:
        seen &= (rel <= 0) | (j < st["prefix"][:, None, None])
    s.masked_fill_(~seen[:, None], -math.inf)
    p, lse = _softmax(s)
    del s
    o = torch.bmm(p.view(n * kv, -1, Lk), v)
    out = {"o": _packed(o.view(n, H, Lq, D), st["q_off"]).to(st["q"].dtype),
           "lse": _packed(lse[..., None], st["q_off"])[..., 0].t().contiguous()}
    if c["kind"] == "attend":
        return out
    do = _padded(st["do"], st["q_off"], Lq).view(n * kv, -1, D)
    dv = torch.bmm(p.view(n * kv, -1, Lk).transpose(1, 2).contiguous(), do)
    dp = torch.bmm(do, v.transpose(1, 2).contiguous()).view(n, H, Lq, Lk)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    del dp, p
    if R:
        # row i of the flipped scores moved i places: a column then holds one distance
        w = Lq + Lk
        turned = torch.cat([ds.flip(-1), ds.new_zeros(n, H, Lq, Lq)], -1).view(n, H, -1)
        by = turned[..., :Lq * (w - 1)].reshape(n, H, Lq, w - 1).sum((0, 2), dtype=torch.float64)
        del turned
        nb, far = _buckets(c)
        at = _bucket((Lk - 1 - torch.arange(w - 1, device=DEV)).clamp(-R, R), nb, far)
        one = (at[None, :] == torch.arange(nb, device=DEV)[:, None]).double()
        out["dtable"] = (one @ by.t().contiguous()).float()
    if t is not None:
        ds *= 1 - t * t
    ds = ds.view(n * kv, -1, Lk)
    dq = torch.bmm(ds, k) * scale
    dk = torch.bmm(ds.transpose(1, 2).contiguous(), q) * scale
    out["dq"] = _packed(dq.view(n, H, Lq, D), st["q_off"]).to(st["q"].dtype)
    out["dk"] = _packed(dk.view(n, kv, Lk, D), st["kv_off"]).to(st["q"].dtype)
    out["dv"] = _packed(dv.view(n, kv, Lk, D), st["kv_off"]).to(st["q"].dtype)
    return out


def _plain_decode(st):
    c = st["case"]
    H, kv, D, R, n = c["heads"], c["kv"], c["dim"], c["bias"], c["docs"]
    k, v = (st[x + "_cache"][st["pages"].long()] if not c["quant"] else
            st[x + "_cache"].view(torch.uint8)[st["pages"].long()].view(torch.float8_e4m3fn) for x in ("k", "v"))
    k, v = k.float(), v.float()
    if c["quant"]:
        k = k * st["k_scale"][st["pages"].long()][..., None]
        v = v * st["v_scale"][st["pages"].long()][..., None]
    L = k.shape[1] * c["page"]
    k, v = (x.transpose(1, 2).reshape(n * kv, L, D) for x in (k, v))
    s = torch.bmm(st["q"].float().view(n * kv, H // kv, D), k.transpose(1, 2).contiguous())
    s = s.view(n, H, L) * (1 / math.sqrt(D))
    if c["cap"]:
        s = c["cap"] * torch.tanh(s / c["cap"])
    j, lens = torch.arange(L, device=DEV)[None, :], st["lens"][:, None]
    if R:
        s = s + st["dist"][:, (j - (lens - 1)).clamp(-R, R) + R].transpose(0, 1)
    s.masked_fill_((j >= lens)[:, None], -math.inf)
    p, lse = _softmax(s)
    o = torch.bmm(p.view(n * kv, H // kv, L), v).view(n, H, D)
    return {"o": o.to(st["q"].dtype), "lse": lse}


def _plain_cache(st):
    c = st["case"]
    page, at = st["slots"] // c["page"], st["slots"] % c["page"]
    for x in ("k", "v"):
        if c["quant"]:
            code, scale = _quantise(st[x])
            held = st[x + "_cache"].view(torch.uint8)
            held[page, :, at] = code.view(torch.uint8)
            st[x + "_scale"][page, :, at] = scale
            back = held[page, :, at].view(torch.float8_e4m3fn).float() * st[x + "_scale"][page, :, at][..., None]
            st[x + "_back"] = back.to(st[x].dtype)
        else:
            st[x + "_cache"][page, :, at] = st[x]
            st[x + "_back"] = st[x + "_cache"][page, :, at]
    return _cache_outputs(st)


def run(st):
    if own:
        return _own_run(st)
    kind = st["case"]["kind"]
    return _plain_decode(st) if kind == "decode" else _plain_cache(st) if kind == "cache" else _plain_attend(st)


# ----------------------------------------------------------------------- work

def work(case):
    D, kv, size = case["dim"], case["kv"], 2
    held = (1 if case.get("quant") else 2) * D + (4 if case.get("quant") else 0)   # a cached row, its scale among it
    if case["kind"] == "cache":
        return {"bytes": case["tokens"] * (2 * kv * (2 * size * D + 2 * held) + 8), "flops": 0}
    H, n = case["heads"], _lengths(case)
    if case["kind"] == "decode":
        return {"bytes": sum(2 * kv * held * x for x in n) + len(n) * H * (2 * size * D + 4),
                "flops": 4 * D * H * sum(n)}
    p, pairs = case["past"], 0
    for x in n:
        if case["causal"]:
            f = min(case["prefix"], x + p)
            pairs += sum(max(f, i + p + 1) for i in range(x))
        else:
            pairs += x * (x + p)
    nq, nk = sum(n), sum(n) + p * len(n)
    rows = (2 * nq * H + 2 * nk * kv) * D * size + 4 * nq * H
    if case["kind"] == "attend":
        return {"bytes": rows + 4 * H * (2 * case["bias"] + 1) * bool(case["bias"]), "flops": 4 * D * H * pairs}
    rows += (2 * nq * H + 2 * nk * kv) * D * size                     # the outputs' gradient, dq, dk, dv
    return {"bytes": rows + (8 * H * _buckets(case)[0] if case["bias"] else 0), "flops": 14 * D * H * pairs}


# ---------------------------------------------------------------------- exact

def _exact_bucket(r, buckets, far):
    half = buckets // 2
    near, d = half // 2, abs(r)
    b = d if d < near else min(half - 1, near + int(math.log(d / near) / math.log(far / near) * (half - near) + 1e-9))
    return b + (half if r > 0 else 0)


def _exact_heads(c, q, k, v, dist, past, prefix):
    """One clip's heads [h][n][d] that share a key head, in 64 bits: (o, lse)."""
    x = torch.matmul(q, k.t()) / math.sqrt(c["dim"])
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    j = torch.arange(k.shape[0], device=DEV)
    r = j[None, :] - torch.arange(past, past + q.shape[1], device=DEV)[:, None]
    if dist is not None:
        R = c["bias"]
        x = x + dist[:, torch.clamp(r, -R, R) + R]
    if c.get("causal"):
        x = torch.where((r > 0) & (j[None, :] >= prefix), torch.full((), -math.inf, device=DEV, dtype=x.dtype), x)
    lse = torch.logsumexp(x, -1)
    return torch.matmul(torch.exp(x - lse[..., None]), v), lse


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    c = case
    if c["kind"] == "cache":
        return _exact_cache(st)
    H, kv, R = c["heads"], c["kv"], c["bias"]
    G = H // kv
    if c["kind"] == "decode":
        o, lse = [], []
        for i, n in enumerate(_lengths(c)):
            pages = st["pages"][i, :-(-n // c["page"])].long()
            k, v = (_exact_rows(st, x, pages)[:, :n] for x in ("k", "v"))
            q = st["q"][i].double().view(kv, G, 1, -1)
            got = [_exact_heads(c, q[h], k[h], v[h], st["dist"][h * G:h * G + G].double() if R else None, n - 1, 0)
                   for h in range(kv)]
            o.append(torch.cat([x[0][:, 0] for x in got]))
            lse.append(torch.cat([x[1][:, 0] for x in got]))
        return {"o": torch.stack(o), "lse": torch.stack(lse)}
    train = c["kind"] == "train"
    q, k, v = (st[x].double() for x in ("q", "k", "v"))
    out = {"o": torch.empty_like(q), "lse": torch.empty(H, q.shape[0], device=DEV, dtype=torch.float64)}
    if train:
        out.update(dq=torch.empty_like(q), dk=torch.empty_like(k), dv=torch.empty_like(v))
    dist = st["dist"].double() if R else None
    ddist = torch.zeros_like(dist) if R and train else None
    for a, b, e, f, p in zip(st["q_at"], st["q_at"][1:], st["kv_at"], st["kv_at"][1:], st["prefix_of"]):
        for h in range(H):
            g = h // G
            x = [q[a:b, h][None].contiguous(), k[e:f, g].contiguous(), v[e:f, g].contiguous(),
                 dist[h:h + 1] if R else None]
            if train:
                x = [None if y is None else y.clone().requires_grad_() for y in x]
            o, lse = _exact_heads(c, *x, (f - e) - (b - a), p)
            out["o"][a:b, h], out["lse"][h, a:b] = o[0].detach(), lse[0].detach()
            if train:
                o.backward(st["do"][a:b, h][None].double())
                out["dq"][a:b, h] = x[0].grad[0]
                for name, y in (("dk", x[1]), ("dv", x[2])):
                    out[name][e:f, g] = y.grad + (out[name][e:f, g] if h % G else 0)
                if R:
                    ddist[h] += x[3].grad[0]
    if R and train:
        nb, far = _buckets(c)
        out["dtable"] = torch.zeros(nb, H, device=DEV, dtype=torch.float64)
        at = torch.tensor([_exact_bucket(r, nb, far) for r in range(-R, R + 1)], device=DEV)
        for b in range(nb):
            out["dtable"][b] = ddist[:, at == b].sum(1)
    return out


def _exact_rows(st, x, pages):
    """The rows [kv][n][d] that a stream's pages hold, in 64 bits."""
    held = st[x + "_cache"]
    if st["case"]["quant"]:
        rows = held.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float().double() \
            * st[x + "_scale"][pages].double()[..., None]
    else:
        rows = held[pages].double()
    return rows.permute(1, 0, 2, 3).flatten(1, 2)


def _exact_cache(st):
    """The values that the cache stands for: rows scaled to the largest code, rounded to 3 bits after the first."""
    c, out = st["case"], {}
    page, at = torch.div(st["slots"], c["page"], rounding_mode="floor"), torch.remainder(st["slots"], c["page"])
    for x in ("k", "v"):
        rows = st[x].double()
        if not c["quant"]:
            out[x] = rows
            held = torch.zeros(st[x + "_cache"].shape, device=DEV, dtype=torch.float64)
            held[page, :, at] = rows
            out[x + "_cache"] = held
            continue
        most = torch.clamp(rows.abs().max(-1, keepdim=True).values, min=TINY)
        scale = most / E4M3_MAX
        y = rows * E4M3_MAX / most
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
        out[x] = torch.round(y / step) * step * scale
        held = torch.zeros(st[x + "_scale"].shape, device=DEV, dtype=torch.float64)
        held[page, :, at] = scale[..., 0]
        out[x + "_scale"] = held
    return out
