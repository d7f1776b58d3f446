"""What is measured of the operators that verify drafted tokens over a KV cache.

Four operators, in the order in which a verification step calls them for a layer (kv_write, tree_attention) and for the
model (token_logprobs, kv_accept):

  kv_write        a fused projection's rows [q | k | v] -> per-head RMSNorm and rotary position on q and k, q in BF16, k and v
                  into the cache, in BF16 or in E4M3 with one F32 scale per position and KV head
  tree_attention  every sequence's rows (one token, a chain or a tree of drafted tokens) attend to the sequence's cached
                  prefix and to the rows of their own sequence that a mask names
  token_logprobs  log-probability of a given token, entropy and the most probable tokens of every row of logits
  kv_accept       the accepted path's cache rows moved up behind the prefix, in every layer

`own` chooses between the framework's calls and the plain form of elementary torch operations.  Lengths, trees and paths of a
case follow from its "mix" number; all values follow from the seed.
"""
import importlib.util
import math
import os
import random
import sys

import torch

own = False

PACKAGE = "ninfer_nvfp4_glm-5.3_flash_2x_dgxspark_b200"
E4M3_MAX = 448.0


def framework():
    """The package's binding, by file path (the folder's name is not a Python identifier)."""
    if "nf_moe" not in sys.modules:
        spec = importlib.util.spec_from_file_location("nf_moe", os.path.join(os.getcwd(), PACKAGE, "nf_moe.py"))
        sys.modules["nf_moe"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules["nf_moe"])
    return sys.modules["nf_moe"]


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    # the decoder stack's attention (32 query heads, 4 KV heads of 128) and vocabulary, unless a case says otherwise
    return [
        # one token of one sequence: the latency of a single user's step
        dict(name="write_1_token", op="write", tokens=1, seqs=1, context=2048, nq=32, nkv=4, dim=128, rotary=128,
             layout="half", scaling="none", kind="e4m3", wide=True, norm=True, mix=1),
        # a padded decode batch of another head layout: part of the head rotated, interleaved pairs, a BF16 cache
        dict(name="write_257_partial_bf16", op="write", tokens=257, seqs=300, context=1000, nq=24, nkv=8, dim=64, rotary=32,
             layout="interleaved", scaling="linear", kind="bf16", wide=True, norm=False, mix=2),
        # a prompt's chunks at far positions of a scaled context, from a BF16 projection
        dict(name="write_8192_yarn", op="write", tokens=8192, seqs=4, context=65536, nq=32, nkv=4, dim=128, rotary=128,
             layout="half", scaling="yarn", kind="e4m3", wide=False, norm=True, mix=3),
        # plain decode of one sequence with a short history
        dict(name="attend_1x1_ctx1000", op="attend", batch=1, nodes=1, context=1000, nq=32, nkv=4, dim=128, kind="e4m3",
             mask="chain", mix=4),
        # the decode batch of the stack's benchmark: 256 sequences with histories of up to 2048
        dict(name="attend_256x1_ctx2048", op="attend", batch=256, nodes=1, context=2048, nq=32, nkv=4, dim=128, kind="e4m3",
             mask="chain", mix=5),
        # small trees of a serving batch, ragged in nodes and in history, BF16 cache
        dict(name="attend_24x16_ctx8191", op="attend", batch=24, nodes=16, context=8191, nq=32, nkv=4, dim=128, kind="bf16",
             mask="tree", mix=6),
        # wide trees over long histories: bound by the products
        dict(name="attend_4x64_ctx65000", op="attend", batch=4, nodes=64, context=65000, nq=32, nkv=4, dim=128, kind="e4m3",
             mask="tree", mix=7),
        # one sampled token's row
        dict(name="logprobs_1", op="logprobs", rows=1, vocab=151552, pad=0, top=20, wide=True, mix=8),
        # the rows of a verification step
        dict(name="logprobs_256", op="logprobs", rows=256, vocab=151552, pad=0, top=5, wide=True, mix=9),
        # a prompt's log-probabilities from BF16 logits with padded rows
        dict(name="logprobs_4001_bf16", op="logprobs", rows=4001, vocab=32003, pad=61, top=1, wide=False, mix=10),
        # one sequence's accepted path in every layer of the stack
        dict(name="accept_1x46", op="accept", layers=46, batch=1, seqs=2, context=2048, nkv=4, dim=128, nodes=16, kind="bf16",
             mix=11),
        # a batch's accepted paths
        dict(name="accept_200x46", op="accept", layers=46, batch=200, seqs=256, context=256, nkv=4, dim=128, nodes=64,
             kind="e4m3", mix=12),
    ]


def log_int(rng, lo, hi):
    """A whole number of [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["write", "attend", "attend", "logprobs", "accept"])
    kind = rng.choice(["e4m3", "bf16"])
    nq, nkv = rng.choice([(32, 4), (32, 8), (16, 16), (28, 4), (12, 1), (24, 8), (40, 8), (10, 2)])
    dim = rng.choice([64, 128])
    mix = rng.randrange(1 << 30)
    if op == "write":
        tokens = log_int(rng, 1, 8192)
        seqs = log_int(rng, 1, 64)
        context = max(log_int(rng, 64, 16384), -(-2 * tokens // seqs))
        while seqs > 1 and seqs * context > 1 << 17:
            seqs //= 2
            context = max(64, -(-2 * tokens // seqs), context // 2)
        return dict(op=op, tokens=tokens, seqs=seqs, context=context, nq=nq, nkv=nkv, dim=dim,
                    rotary=rng.choice([dim, dim, dim // 2, dim // 4, dim - 2]), layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "yarn"]), kind=kind, wide=rng.random() < 0.5,
                    norm=rng.random() < 0.7, mix=mix)
    if op == "attend":
        nodes, context, batch = log_int(rng, 1, 96), log_int(rng, 1, 65000), log_int(rng, 1, 256)
        while batch > 1 and (batch * nkv * context * dim > 1 << 27 or batch * nq * nodes * context > 1 << 28):
            batch = batch * 2 // 3
        while nodes > 1 and batch * nq * nodes * context > 1 << 28:
            nodes //= 2
        return dict(op=op, batch=batch, nodes=nodes, context=max(context, nodes), nq=nq, nkv=nkv, dim=dim, kind=kind,
                    mask=rng.choice(["chain", "tree", "tree", "holes"]), mix=mix)
    if op == "logprobs":
        vocab, rows = log_int(rng, 33, 262144), log_int(rng, 1, 4096)
        while rows * vocab > 1 << 25:
            rows = max(1, rows * 2 // 3)
        return dict(op=op, rows=rows, vocab=vocab, pad=rng.choice([0, 0, 1, 7, 64]), top=rng.choice([0, 1, 2, 5, 8, 20, 32]),
                    wide=rng.random() < 0.5, mix=mix)
    nodes = log_int(rng, 2, 64)
    layers, batch = log_int(rng, 1, 60), log_int(rng, 1, 128)
    context = nodes + log_int(rng, 16, 512)
    while layers > 1 and layers * batch * nkv * dim * context > 1 << 28:
        layers //= 2
    while batch > 1 and layers * batch * nkv * dim * context > 1 << 28:
        batch //= 2
    return dict(op=op, layers=layers, batch=batch, seqs=batch + rng.randrange(3), context=context, nkv=nkv, dim=dim,
                nodes=nodes, kind=kind, mix=mix)


# --------------------------------------------------------------------------------------- lengths, trees and paths of a case
def write_places(case):
    """(sequence, slot, rotary position) of every token: distinct slots; about one token in 50 of a larger batch is padding
    (slot -1); the tokens of a tree share positions, so a position is the slot or a little less."""
    r = random.Random(case["mix"])
    n, seqs, context = case["tokens"], case["seqs"], case["context"]
    per = -(-n // seqs)
    first = [r.randrange(0, context - per + 1) for _ in range(seqs)]
    order = list(range(seqs))
    r.shuffle(order)
    seq = [order[t // per] for t in range(n)]
    slot = [first[seq[t]] + t % per for t in range(n)]
    pos = [max(0, s - r.randrange(0, 3)) for s in slot]
    if n > 16:
        slot = [-1 if r.random() < 0.02 else s for s in slot]
    return seq, slot, pos


def attend_lengths(case):
    """(rows, prefix, cache sequence) of every sequence of the batch."""
    r = random.Random(case["mix"])
    b, nodes, context = case["batch"], case["nodes"], case["context"]
    rows = [nodes if i == 0 else r.randint((nodes + 2) // 3, nodes) for i in range(b)]
    prefix = [r.randint((context - n) // 2, context - n) for n in rows]
    prefix[0] = context - rows[0]
    if b > 3:
        prefix[1] = 0
    seq = list(range(b))
    r.shuffle(seq)
    return rows, prefix, seq


def attend_bits(case):
    """Every row's visible rows of its own sequence, as whole numbers of 64 bits; None for a chain."""
    if case["mask"] == "chain":
        return None
    r = random.Random(case["mix"] + 1)
    words = (case["nodes"] + 63) // 64
    out = []
    for n in attend_lengths(case)[0]:
        bits = []
        for i in range(n):
            above = bits[r.randrange(max(0, i - 9), i)] if i else 0
            bits.append(above | 1 << i)
        if case["mask"] == "holes":  # rows that see none of the drafted rows
            bits = [0 if r.random() < 0.2 else x for x in bits]
        out += [[(x >> 64 * w & (1 << 64) - 1) for w in range(words)] for x in bits]
    return [[x - (1 << 64) if x >> 63 else x for x in row] for row in out]


def accept_paths(case):
    """(prefix, path, length, cache sequence): nodes that grow along the path, as children follow their parents."""
    r = random.Random(case["mix"])
    longest = max(1, min(8, case["nodes"] // 2))
    prefix, path, length = [], [], []
    for _ in range(case["batch"]):
        n = r.randint(1, longest)
        # the nodes behind the first lie above the slots that they move to, as in a wide tree
        p = [0] + sorted(r.sample(range(longest, case["nodes"]), min(n - 1, case["nodes"] - longest)))
        prefix.append(r.randint(0, case["context"] - case["nodes"]))
        length.append(len(p))
        path.append(p + [-1] * (longest - len(p)))
    seq = r.sample(range(case["seqs"]), case["batch"])
    return prefix, path, length, seq


def rope_settings(case):
    """Base, scaling factor and original context of a case's rotary positions."""
    if case["scaling"] == "none":
        return dict(theta=10000.0, factor=1.0, original=0)
    if case["scaling"] == "linear":
        return dict(theta=10000.0, factor=4.0, original=0)
    return dict(theta=500000.0, factor=16.0, original=4096)


# -------------------------------------------------------------------------------------------------------------- prepare
def random_cache(g, shape, kind):
    """Cache contents as earlier steps leave them: about N(0, 1), every E4M3 row with its own scale."""
    x = torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    if kind == "bf16":
        return x, None
    scale = torch.empty(shape[:-1], dtype=torch.float32, device="cuda").uniform_(0.008, 0.024, generator=g)
    return x.mul_(64.0).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    op = case["op"]
    st = dict(case=case, op=op)
    if op == "write":
        heads = case["nq"] + 2 * case["nkv"]
        qkv = randn(case["tokens"], heads * case["dim"]) * (1.0 + randn(1, heads).exp().repeat_interleave(case["dim"], 1))
        st["qkv"] = qkv if case["wide"] else qkv.bfloat16()
        st["q_norm"] = 1.0 + 0.2 * randn(case["dim"]) if case["norm"] else None
        st["k_norm"] = 1.0 + 0.2 * randn(case["dim"]) if case["norm"] else None
        seq, slot, pos = write_places(case)
        st["seq"], st["slot"], st["pos"] = ints(seq), ints(slot), ints(pos)
        shape = (case["seqs"], case["nkv"], case["context"], case["dim"])
        st["k"], st["ks"] = random_cache(g, shape, case["kind"])
        st["v"], st["vs"] = random_cache(g, shape, case["kind"])
        st["q"] = torch.zeros(case["tokens"], case["nq"], case["dim"], dtype=torch.bfloat16, device="cuda")
        if own:
            m, s = framework(), rope_settings(case)
            st["cache"] = m.KvCache(st["k"], st["v"], st["ks"], st["vs"])
            st["rope"] = m.Rope(case["dim"], rotary_dim=case["rotary"], layout=case["layout"], theta=s["theta"],
                                scaling=case["scaling"], factor=s["factor"], original_context=s["original"])
    elif op == "attend":
        rows, prefix, seq = attend_lengths(case)
        start = [0]
        for n in rows:
            start.append(start[-1] + n)
        st["start"], st["prefix"], st["seq"] = ints(start), ints(prefix), ints(seq)
        bits = attend_bits(case)
        st["mask"] = None if bits is None else torch.tensor(bits, dtype=torch.int64, device="cuda")
        st["q"] = (1.5 * randn(start[-1], case["nq"], case["dim"])).bfloat16()
        shape = (case["batch"], case["nkv"], case["context"], case["dim"])
        st["k"], st["ks"] = random_cache(g, shape, case["kind"])
        st["v"], st["vs"] = random_cache(g, shape, case["kind"])
        st["out"] = torch.zeros_like(st["q"])
        if own:
            m = framework()
            st["cache"] = m.KvCache(st["k"], st["v"], st["ks"], st["vs"])
            st["work"] = torch.empty(m.tree_attention_workspace(case["dim"]), dtype=torch.uint8, device="cuda")
    elif op == "logprobs":
        n, v, top = case["rows"], case["vocab"], case["top"]
        # rows between nearly certain and nearly uniform
        x = randn(n, v + case["pad"]) * (0.5 + 4.0 * torch.rand(n, 1, generator=g, device="cuda"))
        x[:, : min(5, v)] += 6.0
        if n > 2:
            x[1, v // 2: v] = -math.inf  # tokens that a grammar rules out
        st["logits"] = (x if case["wide"] else x.bfloat16())[:, :v]
        st["target"] = torch.randint(0, v, (n,), generator=g, device="cuda", dtype=torch.int32)
        f = lambda *s: torch.zeros(*s, dtype=torch.float32, device="cuda")  # noqa: E731
        st["logprob"], st["entropy"], st["top_logprob"] = f(n), f(n), f(n, top)
        st["top"] = torch.zeros(n, top, dtype=torch.int32, device="cuda")
        if own:
            st["work"] = torch.empty(framework().token_logprobs_workspace(n, v, top), dtype=torch.uint8, device="cuda")
    else:
        prefix, path, length, seq = accept_paths(case)
        st["prefix"], st["path"], st["length"], st["seq"] = ints(prefix), ints(path), ints(length), ints(seq)
        shape = (case["layers"], case["seqs"], case["nkv"], case["context"], case["dim"])
        st["k"], st["ks"] = random_cache(g, shape, case["kind"])
        st["v"], st["vs"] = random_cache(g, shape, case["kind"])
        if own:
            m, e = framework(), [None] * case["layers"]
            st["caches"] = m.KvCaches([m.KvCache(*t) for t in zip(st["k"], st["v"], st["ks"] if st["ks"] is not None else e,
                                                                 st["vs"] if st["vs"] is not None else e)])
    return st


# ------------------------------------------------------------------------------------------------------------------ run
def run(st):
    return {"write": run_write, "attend": run_attend, "logprobs": run_logprobs, "accept": run_accept}[st["op"]](st)


def cache_values(x, scale):
    """What a cache's rows stand for, in 32 bits."""
    return x.float() if scale is None else x.float() * scale.unsqueeze(-1)


def frequencies(case):
    """Radians per position of every rotated pair, and the factor on q and k, in 64 bits."""
    s, n = rope_settings(case), case["rotary"]
    f = s["theta"] ** (-2.0 * torch.arange(n // 2, dtype=torch.float64, device="cuda") / n)
    if case["scaling"] == "linear":
        return f / s["factor"], 1.0
    if case["scaling"] == "yarn":
        keep = ((s["original"] * f / (2 * math.pi) - 1.0) / 31.0).clamp(0, 1)  # by turns over the original context, 1 to 32
        return f * keep + f / s["factor"] * (1 - keep), 0.1 * math.log(s["factor"]) + 1.0
    return f, 1.0


def rotated(x, cos, sin, case):
    """Heads x [tokens, heads, dim] turned by the angles [tokens, 1, pairs]."""
    n, half = case["rotary"], case["rotary"] // 2
    a, b = (x[..., :half], x[..., half:n]) if case["layout"] == "half" else (x[..., 0:n:2], x[..., 1:n:2])
    y = x.clone()
    if case["layout"] == "half":
        y[..., :half], y[..., half:n] = a * cos - b * sin, a * sin + b * cos
    else:
        y[..., 0:n:2], y[..., 1:n:2] = a * cos - b * sin, a * sin + b * cos
    return y


def run_write(st):
    case = st["case"]
    if own:
        framework().kv_write(st["cache"], st["rope"], st["qkv"], case["nq"], st["pos"], st["q"], seqs=st["seq"],
                             slots=st["slot"], q_norm=st["q_norm"], k_norm=st["k_norm"])
    else:
        nq, nkv, dim = case["nq"], case["nkv"], case["dim"]
        x = st["qkv"].float().view(case["tokens"], nq + 2 * nkv, dim)
        q, k, v = x[:, :nq], x[:, nq:nq + nkv], x[:, nq + nkv:]
        if case["norm"]:
            q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-5) * st["q_norm"]
            k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + 1e-5) * st["k_norm"]
        f, magnitude = frequencies(case)
        angle = st["pos"].double().unsqueeze(1) * f
        cos, sin = ((magnitude * t).float().unsqueeze(1) for t in (angle.cos(), angle.sin()))
        q, k = rotated(q, cos, sin, case), rotated(k, cos, sin, case)
        st["q"].copy_(q)
        there = (st["slot"] >= 0).nonzero().squeeze(1)
        seq, slot = st["seq"][there].long(), st["slot"][there].long()
        for x, to, scales in ((k[there], st["k"], st["ks"]), (v[there], st["v"], st["vs"])):
            if scales is None:
                to[seq, :, slot] = x.bfloat16()
            else:
                scale = x.abs().amax(-1) / E4M3_MAX
                codes = (x / scale.clamp_min(1e-38).unsqueeze(-1)).to(torch.float8_e4m3fn)
                to.view(torch.uint8)[seq, :, slot] = codes.view(torch.uint8)
                scales[seq, :, slot] = scale
    out = dict(q=st["q"], k=st["k"], v=st["v"])
    return out if st["ks"] is None else dict(out, ks=st["ks"], vs=st["vs"])


def run_attend(st):
    case = st["case"]
    if own:
        framework().tree_attention(st["cache"], st["q"], st["start"], st["prefix"], st["out"], st["work"], cache_seq=st["seq"],
                                   mask=st["mask"])
        return st["out"]
    b, n, nq, nkv, dim, context = (case[x] for x in ("batch", "nodes", "nq", "nkv", "dim", "context"))
    seq = st["seq"].long()
    k = cache_values(st["k"], st["ks"])[seq]
    v = cache_values(st["v"], st["vs"])[seq]
    start, prefix = st["start"].long(), st["prefix"].long()
    rows = start[1:] - start[:-1]
    row = torch.arange(n, device="cuda")
    real = row < rows[:, None]                                     # [b, n]
    index = (start[:-1, None] + row).clamp_max(start[-1] - 1)
    q = st["q"][index].float().view(b, n, nkv, nq // nkv, dim).permute(0, 2, 1, 3, 4).reshape(b, nkv, -1, dim)
    j = torch.arange(context, device="cuda")
    node = j - prefix[:, None]                                     # [b, context]: which of the sequence's rows, if any
    if st["mask"] is None:
        seen = node[:, None] <= row[:, None]
    else:
        at = node.clamp(0, 64 * st["mask"].shape[1] - 1)
        word = st["mask"][index].gather(2, (at // 64)[:, None].expand(-1, n, -1))
        seen = (word >> (at % 64)[:, None]) & 1 > 0
        seen = seen & (node < rows[:, None])[:, None] | (node < 0)[:, None]
    s = q @ k.transpose(2, 3) / math.sqrt(dim)
    s = s.view(b, nkv, n, -1, context).masked_fill_(~seen[:, None, :, None], -math.inf).view(b, nkv, -1, context)
    p = (s - s.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    o = (p @ v) / p.sum(-1, keepdim=True).clamp_min(1e-30)
    o = o.view(b, nkv, n, -1, dim).permute(0, 2, 1, 3, 4).reshape(b, n, nq, dim)
    st["out"][index[real]] = o[real].bfloat16()
    return st["out"]


def run_logprobs(st):
    case = st["case"]
    if own:
        framework().token_logprobs(st["logits"], st["target"], st["logprob"], st["entropy"], st["top"], st["top_logprob"],
                                   st["work"])
    else:
        x = st["logits"].float()
        d = x - x.amax(-1, keepdim=True)
        e = d.exp()
        total = e.sum(-1, dtype=torch.float64)
        log_total = total.log()
        st["logprob"].copy_(d.gather(1, st["target"].long()[:, None])[:, 0] - log_total)
        st["entropy"].copy_(log_total - (e * d.clamp_min(-1e30)).sum(-1, dtype=torch.float64) / total)
        if case["top"]:  # ties go to the lowest index
            value, index = d.sort(dim=-1, descending=True, stable=True)
            st["top"].copy_(index[:, :case["top"]])
            st["top_logprob"].copy_(value[:, :case["top"]] - log_total[:, None])
    out = dict(logprob=st["logprob"], entropy=st["entropy"])
    return dict(out, top=st["top"], top_logprob=st["top_logprob"]) if case["top"] else out


def run_accept(st):
    if own:
        framework().kv_accept(st["caches"], st["prefix"], st["path"], st["length"], cache_seq=st["seq"])
    else:
        path, prefix = st["path"].long(), st["prefix"].long()[:, None]
        j = torch.arange(path.shape[1], device="cuda")
        there = j < st["length"][:, None]
        seq = st["seq"].long()[:, None].expand_as(path)[there]
        source, target = (prefix + path)[there], (prefix + j)[there]
        for x in (st["k"], st["v"], st["ks"], st["vs"]):
            if x is not None:
                x = x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x
                x[:, seq, :, target] = x[:, seq, :, source]
    out = dict(k=st["k"], v=st["v"])
    return out if st["ks"] is None else dict(out, ks=st["ks"], vs=st["vs"])


# ----------------------------------------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "logprobs":
        n = case["rows"] * case["vocab"]
        return dict(bytes=n * (4 if case["wide"] else 2) + case["rows"] * (12 + 8 * case["top"]), flops=5 * n)
    row = case["nkv"] * 2 * (case["dim"] + 4 if case["kind"] == "e4m3" else 2 * case["dim"])  # a position's K and V
    if op == "write":
        q, x = case["nq"] * case["dim"], (case["nq"] + 2 * case["nkv"]) * case["dim"]
        stored = sum(s >= 0 for s in write_places(case)[1])
        return dict(bytes=case["tokens"] * (x * (4 if case["wide"] else 2) + 2 * q + 12) + stored * row,
                    flops=10 * case["tokens"] * x)
    if op == "accept":
        _, path, length, _ = accept_paths(case)
        moved = sum(p[i] != i for p, n in zip(path, length) for i in range(n))
        return dict(bytes=case["layers"] * moved * 2 * row + 4 * sum(length), flops=0)
    rows, prefix, _ = attend_lengths(case)
    bits = attend_bits(case)
    if bits is None:
        pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(rows, prefix))
    else:
        pairs = sum(n * p for n, p in zip(rows, prefix)) + sum(bin(x & (1 << 64) - 1).count("1") for r in bits for x in r)
    return dict(bytes=4 * sum(rows) * case["nq"] * case["dim"] + (sum(rows) + sum(prefix)) * row,
                flops=4 * case["dim"] * case["nq"] * pairs)


# ---------------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    st = prepare(case, seed)
    return {"write": exact_write, "attend": exact_attend, "logprobs": exact_logprobs,
            "accept": exact_accept}[case["op"]](case, st)


def exact_write(case, st):
    nq, nkv, dim, n = case["nq"], case["nkv"], case["dim"], case["rotary"]
    x = st["qkv"].double().view(case["tokens"], -1, dim)
    heads = {"q": x[:, :nq], "k": x[:, nq:nq + nkv], "v": x[:, nq + nkv:]}
    s = rope_settings(case)
    turn = torch.zeros(case["tokens"], n // 2, dtype=torch.float64, device="cuda")
    gain = 1.0
    for i in range(n // 2):
        f = math.exp(-2.0 * i / n * math.log(s["theta"]))
        if case["scaling"] == "linear":
            f /= s["factor"]
        elif case["scaling"] == "yarn":
            turns = s["original"] * f / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - 1.0) / (32.0 - 1.0)))
            f, gain = keep * f + (1 - keep) * f / s["factor"], 1.0 + 0.1 * math.log(s["factor"])
        turn[:, i] = st["pos"].double() * f
    unit = torch.polar(torch.full_like(turn, gain), turn)[:, None]
    for name in ("q", "k"):
        y = heads[name]
        if case["norm"]:
            y = y / (y.pow(2).sum(-1, keepdim=True) / dim + 1e-5).sqrt() * st[name + "_norm"].double()
        y = y.clone()
        if case["layout"] == "half":
            z = torch.complex(y[..., :n // 2], y[..., n // 2:n]) * unit
            y[..., :n // 2], y[..., n // 2:n] = z.real, z.imag
        else:
            z = torch.view_as_complex(y[..., :n].reshape(*y.shape[:2], n // 2, 2).contiguous()) * unit
            y[..., :n] = torch.view_as_real(z).flatten(-2)
        heads[name] = y
    out = dict(q=heads["q"], k=st["k"].double(), v=st["v"].double())
    if st["ks"] is not None:
        out.update(ks=st["ks"].double(), vs=st["vs"].double())
    places = [(t, a, b) for t, (a, b) in enumerate(zip(*write_places(case)[:2])) if b >= 0]
    t, a, b = (torch.tensor(c, dtype=torch.int64, device="cuda") for c in zip(*places)) if places else (None,) * 3
    if places:
        for name in ("k", "v"):
            y = heads[name][t]
            if st["ks"] is not None:
                scale = y.abs().amax(-1) / 448.0
                out[name + "s"][a, :, b] = scale
                y = y / scale.unsqueeze(-1)
            out[name][a, :, b] = y
    return out


def exact_attend(case, st):
    rows, prefix, seq = attend_lengths(case)
    bits = attend_bits(case)
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    group, first = case["nq"] // case["nkv"], 0
    for n, p, c in zip(rows, prefix, seq):
        hidden = torch.zeros(n, p + n, dtype=torch.bool)
        for i in range(n):
            for j in range(n):
                hidden[i, p + j] = j > i if bits is None else not bits[first + i][j // 64] >> j % 64 & 1
        hidden = hidden.cuda()
        for h in range(case["nkv"]):
            k, v = (x[c, h, :p + n].double() if y is None else x[c, h, :p + n].double() * y[c, h, :p + n, None].double()
                    for x, y in ((st["k"], st["ks"]), (st["v"], st["vs"])))
            q = st["q"][first:first + n, h * group:(h + 1) * group].double()
            score = torch.einsum("ngd,jd->ngj", q, k) / case["dim"] ** 0.5
            score = score.masked_fill(hidden[:, None], -math.inf)
            share = torch.softmax(score, -1).nan_to_num(0.0)  # a row that sees nothing has no weights
            out[first:first + n, h * group:(h + 1) * group] = torch.einsum("ngj,jd->ngd", share, v)
        first += n
    return out


def exact_logprobs(case, st):
    rows = {"logprob": [], "entropy": [], "top": None, "top_logprob": []}
    for i in range(0, case["rows"], 256):
        lp = torch.log_softmax(st["logits"][i:i + 256].double(), -1)
        rows["logprob"].append(lp.gather(1, st["target"][i:i + 256].long()[:, None])[:, 0])
        rows["entropy"].append(-(lp.exp() * lp.clamp_min(-1e30)).sum(-1))
        if case["top"]:
            rows["top_logprob"].append(lp.topk(case["top"], -1).values)
    out = dict(logprob=torch.cat(rows["logprob"]), entropy=torch.cat(rows["entropy"]))
    return dict(out, top=None, top_logprob=torch.cat(rows["top_logprob"])) if case["top"] else out


def exact_accept(case, st):
    out = {}
    for name in ("k", "v", "ks", "vs"):
        if st[name] is None:
            continue
        x = out[name] = st[name].double()
        for p, path, n, c in zip(*accept_paths(case)):
            x[:, c, :, p:p + n] = st[name][:, c].double()[:, :, [p + i for i in path[:n]]]
    return out
