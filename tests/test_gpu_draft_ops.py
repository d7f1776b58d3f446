"""The operators of a drafted-token step on the GPU against plain 64-bit
restatements of their formulas.

Tolerances (u = 2^-24 is half a step of F32, h = 2^-8 of BF16, e = 2^-4 of
E4M3, relative to the value):
  kv_write    a normed, rotated value is a handful of F32 operations: the sum
              of squares (a tree over at most 128 values), a quotient, a root,
              two products, the angle (2^-25 of a turn) and the rotation give
              less than 32 u of the head's largest value, 2^-19; the store
              then rounds by h, or by e (2^-10 of the scale below the codes'
              normal range), its scale by 2^-19.
  attention   products of BF16 (E4M3) values are exact in F32 and their sum
              over D <= 128 errs by at most D u sum |q k|, so a score by
              ds = 2^-16 scale max sum |q k|, a weight by 2 ds + 2^-16 (the
              exponential and the running rescale); weights are rounded by h
              before the product with the values, the result by h once more.
  logprobs    the sum of vocab exponentials, at most vocab / 256 + 64 deep,
              errs by (vocab / 256 + 64) u plus 2^-20 for each exponential."""
import numpy as np
import pytest

from helpers import nfm

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
m = nfm()

F32_HEAD = 2.0 ** -19
H_BF16 = 2.0 ** -8
H_E4M3 = 2.0 ** -4


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def make_cache(rng, kind, seqs, nkv, context, dim):
    """Random cache contents and their 64-bit values: (KvCache, k, v)."""
    shape = (seqs, nkv, context, dim)
    x = [torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).bfloat16() for _ in range(2)]
    if kind == "bf16":
        c = m.KvCache(*(t.cuda() for t in x))
        return c, x[0].double().numpy(), x[1].double().numpy()
    s = [torch.from_numpy((0.01 * np.exp(rng.standard_normal(shape[:3]))).astype(np.float32)) for _ in range(2)]
    code = [(t.float() * 60).clamp(-448, 448).to(torch.float8_e4m3fn) for t in x]
    c = m.KvCache(code[0].cuda(), code[1].cuda(), s[0].cuda(), s[1].cuda())
    return c, *(a.float().double().numpy() * b.double().numpy()[..., None] for a, b in zip(code, s))


def cache_host(c):
    """A cache's raw contents on the host."""
    out = []
    for t in c.tensors:
        if t is not None:
            t = t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t.view(torch.int16) if t.dtype == torch.bfloat16 else t
            out.append(t.cpu().numpy().copy())
    return out


# ------------------------------------------------------------------------------------------------------------- kv_write
def exact_head(x, w, eps, rope, pos):
    """One head in 64 bits: RMSNorm (w None: none), then the rotation."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt(np.mean(x * x) + eps) * w.astype(np.float64)
    rd, out = rope["rd"], x.copy()
    f = rope["f"]
    c, s = rope["gain"] * np.cos(pos * f), rope["gain"] * np.sin(pos * f)
    i = np.arange(rd // 2)
    a, b = (i, i + rd // 2) if rope["layout"] == "half" else (2 * i, 2 * i + 1)
    out[a], out[b] = x[a] * c - x[b] * s, x[a] * s + x[b] * c
    return out


def make_rope(dim, rd, layout, scaling):
    theta, factor, original = (500000.0, 16.0, 4096.0) if scaling == "yarn" else (10000.0, 4.0, 0.0)
    f = theta ** (-2.0 * np.arange(rd // 2) / max(rd, 1))
    gain = 1.0
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":
        g = np.clip((original * f / (2 * np.pi) - 1.0) / 31.0, 0, 1)
        f, gain = f * g + f / factor * (1 - g), 0.1 * np.log(factor) + 1
    r = m.Rope(dim, rotary_dim=rd, layout=layout, theta=theta, scaling=scaling, factor=factor, original_context=original)
    return r, dict(rd=rd, f=f, gain=gain, layout=layout)


def check_write(seed, tokens, nq, nkv, dim, kind, wide, layout, rd, scaling, norm, context=300, seqs=3, pad=0, scale=1.0,
                far=1 << 20, call=None):
    rng = np.random.default_rng(seed)
    heads = nq + 2 * nkv
    x = (rng.standard_normal((tokens, heads * dim + pad)) * scale).astype(np.float32)
    xt = torch.from_numpy(x).cuda()
    if not wide:
        xt = xt.bfloat16()
        x = xt.float().cpu().numpy()
    xt = xt[:, :heads * dim]
    qw, kw = ((1 + 0.2 * rng.standard_normal(dim)).astype(np.float32) for _ in range(2))
    c, _, _ = make_cache(rng, kind, seqs, nkv, context, dim)
    before = cache_host(c)
    places = rng.permutation(seqs * context)[:tokens]
    seq, slot = places // context, places % context
    pos = rng.integers(0, far, tokens)
    if tokens > 2:
        slot[1] = -1
    rope, spec = make_rope(dim, rd, layout, scaling)
    q = torch.full((tokens, nq, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    status = ints([0])
    args = dict(seqs=ints(seq), slots=ints(slot), status=status)
    if norm:
        args.update(q_norm=torch.from_numpy(qw).cuda(), k_norm=torch.from_numpy(kw).cuda())
    (call or m.kv_write)(c, rope, xt, nq, ints(pos), q, **args)
    torch.cuda.synchronize()
    assert status.item() == 0
    after = cache_host(c)
    got_q = q.float().cpu().numpy().astype(np.float64)
    touched = np.zeros((seqs, context), bool)
    for t in range(tokens):
        row = x[t, :heads * dim].reshape(heads, dim)
        for h in range(nq):
            want = exact_head(row[h], qw if norm else None, 1e-5, spec, pos[t])
            tol = H_BF16 * np.abs(want) + F32_HEAD * np.abs(want).max() * 2
            assert np.all(np.abs(got_q[t, h] - want) <= tol), (t, h)
        if slot[t] < 0:
            continue
        touched[seq[t], slot[t]] = True
        for g in range(nkv):
            for part, want in ((0, exact_head(row[nq + g], kw if norm else None, 1e-5, spec, pos[t])),
                               (1, row[nq + nkv + g].astype(np.float64))):
                raw = after[part][seq[t], g, slot[t]]
                peak = np.abs(want).max()
                if kind == "bf16":
                    got = torch.from_numpy(raw.copy()).view(torch.bfloat16).double().numpy()
                    tol = H_BF16 * np.abs(want) + 2 * F32_HEAD * peak
                else:
                    s = float(after[2 + part][seq[t], g, slot[t]])
                    assert abs(s - peak / 448) <= 2 * F32_HEAD * peak / 448
                    got = torch.from_numpy(raw.copy()).view(torch.float8_e4m3fn).float().double().numpy() * s
                    tol = H_E4M3 * np.abs(want) + 2.0 ** -10 * s + 4 * F32_HEAD * peak
                assert np.all(np.abs(got - want) <= tol), (t, g, part)
    for a, b in zip(before, after):  # every other row as it was
        a, b = np.moveaxis(a, 2, 1)[~touched], np.moveaxis(b, 2, 1)[~touched]
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8))


@pytest.mark.parametrize("kind", ["e4m3", "bf16"])
@pytest.mark.parametrize("layout, dim, rd, scaling", [
    ("half", 128, 128, "none"), ("interleaved", 128, 128, "yarn"), ("half", 64, 64, "linear"), ("interleaved", 64, 64, "none"),
    ("half", 128, 64, "yarn"), ("half", 128, 126, "none"), ("interleaved", 64, 30, "linear"), ("half", 64, 2, "none"),
    ("half", 128, 0, "none"), ("half", 64, 16, "yarn"), ("interleaved", 128, 32, "none")])
def test_write_layouts(kind, layout, dim, rd, scaling):
    check_write(dim + rd, 9, 4, 2, dim, kind, True, layout, rd, scaling, True)


@pytest.mark.parametrize("tokens, nq, nkv", [(1, 32, 4), (2, 1, 1), (33, 7, 1), (130, 10, 5), (5, 40, 8)])
@pytest.mark.parametrize("kind, wide, norm", [("e4m3", True, True), ("e4m3", False, False), ("bf16", False, True), ("bf16", True, False)])
def test_write_heads_and_types(tokens, nq, nkv, kind, wide, norm):
    check_write(tokens + nq, tokens, nq, nkv, 64 if nq % 2 else 128, kind, wide, "half", 64, "none", norm, pad=16)


@pytest.mark.parametrize("scale", [1e-30, 1e-6, 1e6, 1e15])
def test_write_magnitudes(scale):
    check_write(3, 4, 2, 2, 128, "e4m3", True, "half", 128, "none", False, scale=scale)


def test_write_largest_position():
    check_write(4, 6, 2, 1, 128, "bf16", True, "half", 128, "none", True, far=(1 << 31) - 1)


def test_write_special_rows():
    """A row of zeros has scale 0 and reads back as zeros; a NaN or an infinity makes the row's scale NaN or infinite, so
    that the row reads back as NaN; the rows beside it stay exact."""
    x = torch.zeros(4, 4 * 64, device="cuda")
    x[1], x[3] = 1.0, 2.0
    x[1, 2 * 64 + 5], x[2, 3 * 64 + 7] = float("nan"), float("inf")
    k = torch.zeros(1, 1, 4, 64, dtype=torch.float8_e4m3fn, device="cuda")
    c = m.KvCache(k, k.clone(), *(torch.full((1, 1, 4), 9.0, device="cuda") for _ in range(2)))
    q = torch.empty(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    m.kv_write(c, m.Rope(64), x, 2, ints([0] * 4), q, seqs=ints([0] * 4), slots=ints(range(4)))
    back = [c.tensors[i].float()[0, 0] * c.tensors[i + 2][0, 0, :, None] for i in range(2)]
    assert torch.all(back[0][0] == 0) and torch.all(back[1][0] == 0) and c.tensors[2][0, 0, 0] == 0
    assert torch.all(back[0][1].isnan()) and torch.all(back[1][1] == 1)
    assert torch.all(back[0][2] == 0) and torch.all(back[1][2].isnan())
    assert torch.all(back[0][3] == 2) and torch.all(back[1][3] == 2)


def test_write_defaults_and_bad_indices():
    """Without seqs and slots token t goes to position pos[t] of sequence t; a token with an index outside is left out, gets a
    q of NaN and sets the status; a padding slot only skips the cache."""
    rng = np.random.default_rng(8)
    x = torch.from_numpy(rng.standard_normal((3, 4 * 64)).astype(np.float32)).cuda()
    c, _, _ = make_cache(rng, "bf16", 3, 1, 10, 64)
    old = c.tensors[1].clone()
    q = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    m.kv_write(c, m.Rope(64), x, 2, ints([0, 9, 4]), q)
    for t, p in enumerate((0, 9, 4)):
        assert torch.equal(c.tensors[1][t, 0, p], x[t, 192:].bfloat16())
        old[t, 0, p] = x[t, 192:].bfloat16()
    assert torch.equal(c.tensors[1], old) and not q.isnan().any()
    for pos, seq, slot in ((-1, 0, 0), (0, 3, 0), (0, -1, 0), (0, 0, 10), (0, 0, -2)):
        status = ints([0])
        m.kv_write(c, m.Rope(64), x[:1], 2, ints([pos]), q[:1], seqs=ints([seq]), slots=ints([slot]), status=status)
        assert status.item() != 0 and q[:1].isnan().all()
        m.kv_write(c, m.Rope(64), x[:1], 2, ints([pos]), q[:1], seqs=ints([seq]), slots=ints([slot]))  # without a status
        assert torch.equal(c.tensors[1], old)
    status = ints([0])
    m.kv_write(c, m.Rope(64), x[:1], 2, ints([3]), q[:1], seqs=ints([99]), slots=ints([-1]), status=status)
    assert status.item() == 0 and not q[:1].isnan().any() and torch.equal(c.tensors[1], old)


def test_write_refuses_tensors():
    rng = np.random.default_rng(1)
    c, _, _ = make_cache(rng, "bf16", 2, 1, 8, 64)
    q = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    x = torch.zeros(2, 256, device="cuda")
    r, p = m.Rope(64), ints([0, 0])
    for bad in (lambda: m.kv_write(c, r, x[:, :192], 2, p, q), lambda: m.kv_write(c, r, x.double(), 2, p, q),
                lambda: m.kv_write(c, r, x.cpu(), 2, p, q), lambda: m.kv_write(c, r, x, 2, p[:1], q),
                lambda: m.kv_write(c, r, x, 2, p.long(), q), lambda: m.kv_write(c, r, x, 2, p, q[:1]),
                lambda: m.kv_write(c, m.Rope(128), x, 2, p, q), lambda: m.kv_write(c, r, x.t().contiguous().t(), 2, p, q),
                lambda: m.kv_write(c, r, torch.zeros(3, 256, device="cuda"), 2, ints([0] * 3), torch.cat([q, q])),
                lambda: m.KvCache(c.tensors[0], c.tensors[1][:1]), lambda: m.KvCache(c.tensors[0], c.tensors[1], x, x),
                lambda: m.KvCache(c.tensors[0][:, :, ::2], c.tensors[1][:, :, ::2]), lambda: m.KvCache(x, x)):
        with pytest.raises(m.NfError):
            bad()


# ------------------------------------------------------------------------------------------------------- tree attention
def tree_words(rng, rows, words, kind):
    """Mask words of every row of one sequence, and the same as truth values [rows, 64 words]."""
    see = np.zeros((rows, 64 * words), bool)
    for i in range(rows):
        if kind == "tree" and i:
            see[i] = see[rng.integers(max(0, i - 7), i)]
        if kind in ("tree", "holes") and i < 64 * words:
            see[i, i] = True
        if kind == "any":
            see[i] = rng.random(64 * words) < 0.4  # rows behind the sequence's among them
        if kind == "holes" and rng.random() < 0.4:
            see[i] = False
    bits = see.reshape(rows, words, 64).astype(np.uint64) << np.arange(64, dtype=np.uint64)
    return bits.sum(-1, dtype=np.uint64).view(np.int64), see


def exact_attention(q, k, v, see, scale):
    """q [G, D] of one row and KV head over the keys named by `see`: (result, tolerance)."""
    k, v = k[see], v[see]
    if not len(k):
        return np.zeros_like(q), np.zeros_like(q)
    s = q @ k.T * scale
    p = np.exp(s - s.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    out = p @ v
    ds = 2.0 ** -16 * abs(scale) * (np.abs(q) @ np.abs(k).T).max(1, keepdims=True)
    return out, H_BF16 * np.abs(out) + (H_BF16 + 2 * ds + 2.0 ** -16) * (p @ np.abs(v))


def check_attention(seed, rows, prefix, nq, nkv, dim, kind, mask=None, words=1, seq=None, seqs=None, context=None, scale=None,
                    spread=1.0, extra=3, behind=None, call=None, work=None):
    rng = np.random.default_rng(seed)
    b = len(rows)
    context = context or max(p + n for p, n in zip(prefix, rows))
    seqs = seqs or b
    c, k, v = make_cache(rng, kind, seqs, nkv, context, dim)
    place = seq if seq is not None else list(range(b))
    if behind is not None:  # what lies behind a sequence's rows must not matter
        for i in range(b):
            for t in c.tensors[:2]:
                end = prefix[i] + rows[i]
                if t.dtype == torch.float8_e4m3fn:
                    t.view(torch.uint8)[place[i], :, end:] = 0x7f
                else:
                    t[place[i], :, end:] = behind
            for t in c.tensors[2:]:
                if t is not None:
                    t[place[i], :, end:] = behind
    total = sum(rows)
    q = torch.from_numpy((spread * rng.standard_normal((total + extra, nq, dim))).astype(np.float32)).bfloat16()
    start = np.concatenate([[0], np.cumsum(rows)])
    bits, see = None, []
    if mask is not None:
        pairs = [tree_words(rng, n, words, mask) for n in rows]
        bits = torch.from_numpy(np.concatenate([p[0] for p in pairs] + [np.full((extra, words), -1, np.int64)])).cuda()
        see = [p[1] for p in pairs]
    out = torch.full((total + extra, nq, dim), 5.0, dtype=torch.bfloat16, device="cuda")
    work = torch.empty(m.tree_attention_workspace(dim), dtype=torch.uint8, device="cuda") if work is None else work
    status = ints([0])
    (call or m.tree_attention)(c, q.cuda(), ints(start), ints(prefix), out, work, mask=bits, scale=scale, status=status,
                               cache_seq=None if seq is None else ints(seq))
    torch.cuda.synchronize()
    assert status.item() == 0
    got = out.double().cpu().numpy()
    assert np.all(got[total:] == 5.0), "rows behind the last sequence"
    qd, G = q.double().numpy(), nq // nkv
    for i in range(b):
        n, p = rows[i], prefix[i]
        for r in range(n):
            vis = np.ones(p + n, bool)
            if mask is None:
                vis[p + r + 1:] = False
            else:
                vis[p:] = np.concatenate([see[i][r], np.zeros(n, bool)])[:n]
            for g in range(nkv):
                want, tol = exact_attention(qd[start[i] + r, g * G:(g + 1) * G], k[place[i], g, :p + n], v[place[i], g, :p + n],
                                            vis, scale if scale is not None else dim ** -0.5)
                err = np.abs(got[start[i] + r, g * G:(g + 1) * G] - want)
                assert np.all(err <= tol), (i, r, g, float(err.max()), float(tol.flat[err.argmax()]))
    return out


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("length", [0, 1, 2, 31, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300, 1000])
def test_attention_one_row(kind, dim, length):
    check_attention(length, [1], [length], 8, 1, dim, kind)


@pytest.mark.parametrize("nq, nkv", [(1, 1), (3, 1), (8, 8), (32, 4), (10, 5), (28, 4), (16, 1), (17, 1), (48, 3), (128, 1), (100, 1)])
@pytest.mark.parametrize("kind, dim", [("bf16", 128), ("e4m3", 64), ("e4m3", 128)])
def test_attention_head_layouts(nq, nkv, kind, dim):
    check_attention(nq + dim, [3, 1], [200, 70], nq, nkv, dim, kind)


@pytest.mark.parametrize("kind, dim", [("bf16", 128), ("bf16", 64), ("e4m3", 128)])
@pytest.mark.parametrize("mask", [None, "tree", "holes", "any"])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 33, 63, 64])
def test_attention_trees(kind, dim, mask, n):
    check_attention(n, [n, 2, n], [140, 0, 61], 8, 1, dim, kind, mask=mask)


@pytest.mark.parametrize("words, n", [(2, 65), (2, 128), (3, 130), (1, 100), (4, 256)])
def test_attention_wide_masks(words, n):
    """Several mask words; with one word a row sees nothing of the rows from 64 on."""
    check_attention(words, [n, 5], [30, 99], 4, 2, 64, "e4m3", mask="any", words=words)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_attention_prompt_chunk(kind):
    """A chain longer than any tile, from an empty cache and behind a prefix."""
    check_attention(5, [300, 140], [0, 150], 4, 2, 128, kind)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_attention_ragged_batch(kind):
    rng = np.random.default_rng(12)
    b = 37
    rows = rng.integers(1, 9, b).tolist()
    rows[3] = 0  # a sequence without rows
    prefix = rng.integers(0, 400, b).tolist()
    prefix[5] = 0
    check_attention(13, rows, prefix, 8, 2, 128, kind, mask="tree", seq=rng.permutation(b + 3)[:b].tolist(), seqs=b + 3,
                    context=450, behind=float("nan"))


@pytest.mark.parametrize("kind, dim", [("bf16", 128), ("e4m3", 128), ("e4m3", 64), ("bf16", 64)])
def test_attention_long_split(kind, dim):
    """One sequence over every SM, and a second short one: the parts of a row are joined."""
    check_attention(21, [2, 1], [50_001, 3], 8, 1, dim, kind, mask="tree")
    check_attention(22, [20], [30_000], 16, 2, dim, kind, mask="tree")


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("spread, scale", [(8.0, 1.0), (1.0, 0.0), (30.0, -0.5), (1e-3, None)])
def test_attention_score_ranges(kind, spread, scale):
    """Scores of some hundreds (one key takes all), equal scores, a negative scale."""
    check_attention(31, [5], [333], 8, 1, 128, kind, spread=spread, scale=scale)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("n, length", [(1, 5), (1, 129), (7, 64), (20, 200)])
def test_attention_ignores_what_lies_behind(kind, n, length):
    """NaN and infinities behind a sequence's rows reach nothing."""
    for bad in (float("nan"), float("inf")):
        check_attention(41, [n, n], [length, 3], 8, 1, 128, kind, mask="tree", behind=bad, context=length + n + 300)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_attention_nan_in_an_unseen_row(kind):
    """A NaN in the key or the value of a drafted row reaches only the rows that see it."""
    rng = np.random.default_rng(51)
    c, _, _ = make_cache(rng, kind, 1, 1, 80, 128)
    for part in (0, 1):
        t = c.tensors[part]
        if kind == "bf16":
            t[0, 0, 62] = float("nan")
        else:
            t.view(torch.uint8)[0, 0, 62] = 0x7f
    q = torch.from_numpy(rng.standard_normal((4, 8, 128)).astype(np.float32)).bfloat16().cuda()
    bits = torch.tensor([[1], [3], [5], [13]], dtype=torch.int64, device="cuda")  # row 2 lies at position 62
    out, work = torch.zeros_like(q), torch.empty(m.tree_attention_workspace(128), dtype=torch.uint8, device="cuda")
    m.tree_attention(c, q, ints([0, 4]), ints([60]), out, work, mask=bits)
    bad = out.isnan().flatten(1)
    assert not bad[:2].any() and bad[2:].all()


def test_attention_bad_sequences():
    """A sequence whose indices lie outside gives NaN and sets the status; its neighbours are exact."""
    rng = np.random.default_rng(61)
    c, _, _ = make_cache(rng, "e4m3", 3, 2, 50, 64)
    q = torch.from_numpy(rng.standard_normal((6, 4, 64)).astype(np.float32)).bfloat16().cuda()
    work = torch.empty(m.tree_attention_workspace(64), dtype=torch.uint8, device="cuda")
    good = torch.zeros_like(q)
    m.tree_attention(c, q, ints([0, 2, 4, 6]), ints([10, 20, 30]), good, work)
    for prefix, seq in (([10, -1, 30], [0, 1, 2]), ([10, 49, 30], [0, 1, 2]), ([10, 20, 30], [0, 3, 2]), ([10, 20, 30], [0, -1, 2]),
                        ([10, 2 ** 31 - 1, 30], [0, 1, 2])):
        out, status = torch.zeros_like(q), ints([0])
        m.tree_attention(c, q, ints([0, 2, 4, 6]), ints(prefix), out, work, cache_seq=ints(seq), status=status)
        assert status.item() != 0 and out[2:4].isnan().all()
        assert torch.equal(out[:2], good[:2]) and torch.equal(out[4:], good[4:])
        m.tree_attention(c, q, ints([0, 2, 4, 6]), ints(prefix), out, work, cache_seq=ints(seq))
    out = torch.zeros_like(q)  # row_start outside the rows: clamped
    m.tree_attention(c, q, ints([-3, 2, 4, 99]), ints([10, 20, 30]), out, work)
    assert torch.equal(out, good)


def test_attention_repeats_bit_for_bit():
    rng = np.random.default_rng(71)
    c, _, _ = make_cache(rng, "e4m3", 5, 2, 3000, 128)
    q = torch.from_numpy(rng.standard_normal((5 * 9, 16, 128)).astype(np.float32)).bfloat16().cuda()
    start, prefix = ints(range(0, 46, 9)), ints([2991, 7, 1500, 0, 129])
    work = torch.empty(m.tree_attention_workspace(128), dtype=torch.uint8, device="cuda")
    outs = []
    for _ in range(3):
        work.random_(0, 256)  # the workspace's contents do not matter
        outs.append(torch.empty_like(q))
        m.tree_attention(c, q, start, prefix, outs[-1], work)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("rows", [1, 20, 48])
@pytest.mark.parametrize("course", ["rising", "falling", "late", "flat"])
def test_attention_courses_of_the_maximum(kind, rows, course):
    """Scores that rise or fall along the keys by hundreds, so that the running maximum moves in every tile or never."""
    nq, nkv, dim, prefix = 8, 1, 128, 1000
    rng = np.random.default_rng(rows)
    c, k, v = make_cache(rng, kind, 1, nkv, prefix + rows, dim)
    at = np.arange(prefix + rows) / (prefix + rows)
    gain = {"rising": at, "falling": 1 - at, "late": (at > 0.9) * 1.0, "flat": 0 * at}[course]
    u = np.sign(rng.standard_normal(dim))
    # every key: a multiple of u (exact in both types) instead of its random row
    want = np.round(gain * 16) / 16
    if kind == "bf16":
        c.tensors[0][0, 0] = torch.from_numpy(want[:, None] * u).bfloat16().cuda()
    else:
        c.tensors[0][0, 0] = torch.from_numpy(want[:, None] * u).float().cuda().to(torch.float8_e4m3fn)
        c.tensors[2].fill_(1.0)
    k = c.tensors[0][0, 0].float().double().cpu().numpy()
    q = torch.from_numpy(np.tile(2.5 * u, (rows, nq, 1)) + 0.1 * rng.standard_normal((rows, nq, dim))).bfloat16()
    out = torch.empty(rows, nq, dim, dtype=torch.bfloat16, device="cuda")
    work = torch.empty(m.tree_attention_workspace(dim), dtype=torch.uint8, device="cuda")
    m.tree_attention(c, q.cuda(), ints([0, rows]), ints([prefix]), out, work, scale=1.0)
    got = out.double().cpu().numpy()
    for r in (0, rows // 2, rows - 1):
        w, tol = exact_attention(q[r].double().numpy(), k, v[0, 0], np.arange(prefix + rows) <= prefix + r, 1.0)
        err = np.abs(got[r] - w)
        assert np.all(err <= tol), (r, float(err.max()), float(tol.flat[err.argmax()]))


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("batch, nodes", [(32, 1), (24, 2), (12, 16)])
def test_attention_from_cold_memory(kind, batch, nodes):
    """Long caches that the L2 does not hold, whose loads land in any order."""
    nq, nkv, dim, context = 32, 4, 128, 4000
    g = torch.Generator(device="cuda").manual_seed(batch)
    x = [torch.randn(batch, nkv, context, dim, device="cuda", generator=g) for _ in range(2)]
    if kind == "bf16":
        c = m.KvCache(*(t.bfloat16() for t in x))
        k, v = (t.double() for t in c.tensors[:2])
    else:
        s = [0.01 * torch.rand(batch, nkv, context, device="cuda", generator=g) for _ in x]
        c = m.KvCache(*((60 * t).clamp(-448, 448).to(torch.float8_e4m3fn) for t in x), *s)
        k, v = (t.float().double() * f.double()[..., None] for t, f in zip(c.tensors[:2], s))
    q = torch.randn(batch * nodes, nq, dim, device="cuda", generator=g).bfloat16()
    lengths = [context - nodes - 37 * i for i in range(batch)]
    start, prefix = ints(range(0, batch * nodes + 1, nodes)), ints(lengths)
    work = torch.empty(m.tree_attention_workspace(dim), dtype=torch.uint8, device="cuda")
    flush = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")
    outs = []
    for _ in range(10):
        flush.zero_()
        outs.append(torch.empty_like(q))
        m.tree_attention(c, q, start, prefix, outs[-1], work)
    torch.cuda.synchronize()
    assert all(torch.equal(outs[0], o) for o in outs[1:])
    for i in (0, batch // 2, batch - 1):
        for r in {0, nodes - 1}:
            for h in (0, nkv - 1):
                heads = slice(h * nq // nkv, (h + 1) * nq // nkv)
                want, tol = exact_attention(q[i * nodes + r, heads].double().cpu().numpy(), k[i, h].cpu().numpy(),
                                            v[i, h].cpu().numpy(), np.arange(context) <= lengths[i] + r, dim ** -0.5)
                err = np.abs(outs[0][i * nodes + r, heads].double().cpu().numpy() - want)
                assert np.all(err <= tol), (i, r, h, float(err.max()))


@pytest.mark.parametrize("nodes", [1, 24])
def test_attention_from_two_threads_on_two_streams(nodes):
    """Calls in flight at the same time, with a workspace each."""
    import threading
    rng = np.random.default_rng(nodes)
    c, _, _ = make_cache(rng, "e4m3", 6, 2, 900, 128)
    q = [torch.from_numpy(rng.standard_normal((6 * nodes, 16, 128)).astype(np.float32)).bfloat16().cuda() for _ in range(2)]
    start, prefix = ints(range(0, 6 * nodes + 1, nodes)), ints([876, 3, 500, 0, 129, 800])
    want = [torch.empty_like(x) for x in q]
    for x, o in zip(q, want):
        m.tree_attention(c, x, start, prefix, o, torch.empty(m.tree_attention_workspace(128), dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    bad = []

    def work(i):
        s = torch.cuda.Stream()
        w = torch.empty(m.tree_attention_workspace(128), dtype=torch.uint8, device="cuda")
        o = [torch.empty_like(q[i]) for _ in range(20)]
        torch.cuda.synchronize()
        for x in o:
            m.tree_attention(c, q[i], start, prefix, x, w, stream=s.cuda_stream)
        s.synchronize()
        bad.extend(1 for x in o if not torch.equal(x, want[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_attention_refuses_tensors():
    rng = np.random.default_rng(1)
    c, _, _ = make_cache(rng, "bf16", 2, 2, 8, 64)
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device="cuda")
    w = torch.empty(m.tree_attention_workspace(64), dtype=torch.uint8, device="cuda")
    s, p = ints([0, 1, 3]), ints([0, 0])
    for bad in (lambda: m.tree_attention(c, q, s, p, q[:1], w), lambda: m.tree_attention(c, q.float(), s, p, q, w),
                lambda: m.tree_attention(c, q[:, :3], s, p, q, w), lambda: m.tree_attention(c, q, s, p[:1], q, w),
                lambda: m.tree_attention(c, q, s, p, q, w[:16]), lambda: m.tree_attention(c, q, s, p, q, w.cpu()),
                lambda: m.tree_attention(c, q, s, p, q, w, mask=s), lambda: m.tree_attention(c, q, s[:0], p, q, w),
                lambda: m.tree_attention(c, q, s, p, q, w, mask=torch.zeros(2, 1, dtype=torch.int64, device="cuda")),
                lambda: m.tree_attention(c, q[..., :32], s, p, q, w)):
        with pytest.raises(m.NfError):
            bad()


# ------------------------------------------------------------------------------------------------------- log-probabilities
def run_logprobs(x, target, top, work=None):
    n, v = x.shape
    lp, en, tl = (torch.full(s, 9.0, device="cuda") for s in ((n,), (n,), (n, top)))
    ti = torch.full((n, top), -9, dtype=torch.int32, device="cuda")
    work = torch.empty(m.token_logprobs_workspace(n, v, top), dtype=torch.uint8, device="cuda") if work is None else work
    work.random_(0, 256)
    m.token_logprobs(x, target, lp, en, ti if top else None, tl if top else None, work)
    torch.cuda.synchronize()
    return lp.double().cpu().numpy(), en.double().cpu().numpy(), ti.cpu().numpy(), tl.double().cpu().numpy()


def order(row):
    """Indices by falling logit, the lower first among equals, NaN last."""
    key = np.where(np.isnan(row), -np.inf, row)
    return np.lexsort((np.arange(len(row)), np.isnan(row), -key))


def check_logprobs(x, target, top):
    lp, en, ti, tl = run_logprobs(x, target, top)
    xd, t = x.float().double().cpu().numpy(), target.cpu().numpy()
    for r, row in enumerate(xd):
        v = len(row)
        assert np.array_equal(ti[r], order(row)[:top]), r
        if not np.isfinite(row.max()):
            assert np.isnan(lp[r]) and np.isnan(en[r]) and np.isnan(tl[r]).all()
            continue
        d = row - row.max()
        with np.errstate(divide="ignore"):
            full = d - np.log(np.exp(d).sum())
        p = np.exp(full)
        depth = (v / 256 + 64) * 2.0 ** -24 + 2.0 ** -20
        tol = lambda a: depth + 2.0 ** -21 * np.abs(a)  # noqa: E731
        ok = 0 <= t[r] < v
        assert np.isnan(lp[r]) if not ok else lp[r] == full[t[r]] or abs(lp[r] - full[t[r]]) <= tol(full[t[r]]), r
        dz = np.where(p > 0, d, 0)
        assert abs(en[r] + (p * np.where(p > 0, full, 0)).sum()) <= 2 * depth * (1 + (p * np.abs(dz)).sum() + abs(np.log(v))), r
        want = full[ti[r]]
        same = (tl[r] == want) | (np.abs(tl[r] - np.where(np.isfinite(want), want, 0)) <= tol(np.where(np.isfinite(want), want, 0)))
        assert same.all(), r


def logits(rng, rows, vocab, wide, pad=0, ties=False, spread=3.0):
    x = torch.from_numpy((spread * rng.standard_normal((rows, vocab + pad))).astype(np.float32))
    if ties:
        x = x.round()
    return (x if wide else x.bfloat16()).cuda()[:, :vocab]


@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("rows, vocab, top, pad", [
    (1, 1, 1, 0), (1, 2, 2, 1), (3, 31, 20, 3), (2, 33, 32, 0), (5, 1000, 1, 0), (4, 1023, 32, 2), (3, 4097, 8, 7), (2, 32003, 5, 61),
    (1, 151552, 20, 0), (7, 50257, 0, 1), (300, 513, 3, 5)])
def test_logprobs(wide, rows, vocab, top, pad):
    rng = np.random.default_rng(vocab + top)
    check_logprobs(logits(rng, rows, vocab, wide, pad), torch.from_numpy(rng.integers(0, vocab, rows)).int().cuda(), top)


@pytest.mark.parametrize("wide", [True, False])
def test_logprobs_ties_and_order(wide):
    """Equal logits go to the lower index (-0 equals +0), also when they fall on both sides of the cut."""
    rng = np.random.default_rng(3)
    x = logits(rng, 6, 20000, wide, ties=True, spread=1.0)
    x[0] = 0.0
    x[1, ::2], x[1, 1::2] = -0.0, 0.0
    x[2, -1], x[2, 5000], x[2, 0] = 9.0, 9.0, 9.0
    x[3] = torch.arange(20000, device="cuda").flip(0).float().to(x.dtype)   # falling: the first are the greatest
    x[4] = torch.arange(20000, device="cuda").float().to(x.dtype)           # rising: the last are
    check_logprobs(x, ints([0, 1, 2, 19999, 19999, 7]), 32)


@pytest.mark.parametrize("wide", [True, False])
def test_logprobs_special_rows(wide):
    rng = np.random.default_rng(4)
    x = logits(rng, 9, 3001, wide)
    inf = float("inf")
    x[0, 17] = float("nan")
    x[1] = -inf
    x[2, 3000] = inf
    x[3, 1:] = -inf                    # one token left: log-probability 0, entropy 0
    x[4, 100:] = -inf                  # more top tokens than finite logits with top 32 over 100: none; target masked
    x[5, 20:] = -inf
    x[6] = float("nan")
    x[7] = 1000.0                      # uniform, far from zero
    x[8, 5] = torch.finfo(x.dtype).max
    target = ints([17, 0, 3000, 0, 200, 7, 1, 3, 5])
    check_logprobs(x, target, 32)
    check_logprobs(x, ints([-1, 3001, -(2 ** 31), 2 ** 31 - 1, 3000, 0, 0, 0, 6]), 5)


def test_logprobs_far_masks():
    """A mask by the type's lowest value behaves as a mask by -infinity."""
    rng = np.random.default_rng(5)
    x = logits(rng, 2, 5000, True)
    x[:, 7:] = torch.finfo(torch.float32).min
    check_logprobs(x, ints([3, 9]), 8)


def test_logprobs_optional_outputs():
    rng = np.random.default_rng(6)
    x = logits(rng, 3, 700, True)
    work = torch.empty(m.token_logprobs_workspace(3, 700, 4), dtype=torch.uint8, device="cuda")
    lp, en = torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda")
    ti, tl = torch.zeros(3, 4, dtype=torch.int32, device="cuda"), torch.zeros(3, 4, device="cuda")
    m.token_logprobs(x, ints([1, 2, 3]), lp, en, ti, tl, work)
    lp2, tl2 = torch.zeros_like(lp), torch.zeros_like(tl)
    m.token_logprobs(x, ints([1, 2, 3]), lp2, None, None, None, work)
    m.token_logprobs(x, None, None, None, ti, tl2, work)
    assert torch.equal(lp, lp2) and torch.equal(tl, tl2)
    for bad in (lambda: m.token_logprobs(x, None, lp, en, ti, tl, work), lambda: m.token_logprobs(x.double(), None, None, en, ti, tl, work),
                lambda: m.token_logprobs(x, None, None, en, ti, None, work), lambda: m.token_logprobs(x, None, None, en[:2], ti, tl, work),
                lambda: m.token_logprobs(x.t(), None, None, en, ti, tl, work), lambda: m.token_logprobs(x, None, None, en, ti, tl, work[:0])):
        with pytest.raises(m.NfError):
            bad()


# ------------------------------------------------------------------------------------------------------------- kv_accept
@pytest.mark.parametrize("kind, dim", [("bf16", 128), ("bf16", 64), ("e4m3", 128), ("e4m3", 64)])
@pytest.mark.parametrize("layers, batch, longest", [(1, 1, 1), (3, 4, 7), (70, 2, 5), (2, 30, 24)])
def test_accept(kind, dim, layers, batch, longest):
    rng = np.random.default_rng(layers + batch)
    context, seqs = 90, batch + 2
    caches = [make_cache(rng, kind, seqs, 2, context, dim)[0] for _ in range(layers)]
    before = [cache_host(c) for c in caches]
    prefix = rng.integers(0, context - 2 * longest, batch)
    length = rng.integers(0, longest + 1, batch)
    length[0] = longest
    path = np.full((batch, longest), -5)
    for i in range(batch):  # rising, often overlapping the slots they move to
        path[i, :length[i]] = np.sort(rng.permutation(2 * longest)[:length[i]])
    seq = rng.permutation(seqs)[:batch]
    status = ints([0])
    m.kv_accept(m.KvCaches(caches), ints(prefix), ints(path), ints(length), cache_seq=ints(seq), status=status)
    torch.cuda.synchronize()
    assert status.item() == 0
    for c, old in zip(caches, before):
        for a, b in zip(old, cache_host(c)):
            want = a.copy()
            for i in range(batch):
                for j in range(length[i]):
                    want[seq[i], :, prefix[i] + j] = a[seq[i], :, prefix[i] + path[i, j]]
            assert np.array_equal(want.view(np.uint8), b.view(np.uint8))


def test_accept_bad_paths():
    """A path that does not rise or leaves the cache, a prefix or sequence outside: the sequence stays, the status tells; the
    other sequences move."""
    rng = np.random.default_rng(9)
    for prefix, path, length, seq in ((50, [2, 1], 2, 1), (50, [1, 1], 2, 1), (50, [0, 10], 2, 1), (-1, [0, 1], 2, 1),
                                      (61, [0, 1], 1, 1), (50, [-1, 2], 2, 1), (50, [1, 2], 3, 1), (50, [1, 2], -1, 1),
                                      (50, [1, 2], 2, 9), (50, [1, 2], 2, -1), (2 ** 31 - 1, [1, 2], 2, 1)):
        c, _, _ = make_cache(rng, "e4m3", 3, 1, 60, 64)
        before, status = cache_host(c), ints([0])
        m.kv_accept(m.KvCaches([c]), ints([prefix, 10]), ints([path, [3, 4]]), ints([length, 2]), cache_seq=ints([seq, 2]),
                    status=status)
        after = cache_host(c)
        assert status.item() != 0
        for a, b in zip(before, after):
            a[2, :, 10], a[2, :, 11] = a[2, :, 13].copy(), a[2, :, 14].copy()
            assert np.array_equal(a.view(np.uint8), b.view(np.uint8))


def test_accept_more_sequences_than_a_grid_has_rows():
    n = 70000
    k = torch.arange(n, device="cuda").remainder(251).to(torch.int16)[:, None, None, None].repeat(1, 1, 2, 64)
    k[:, :, 1] += 1000
    c = m.KvCache(k, k.clone())
    m.kv_accept(m.KvCaches([c]), ints(np.zeros(n)), ints(np.ones((n, 1))), ints(np.ones(n)))
    torch.cuda.synchronize()
    assert all(torch.equal(t[:, :, 0], t[:, :, 1]) and torch.equal(t[:, 0, 1, 5], k[:, 0, 1, 5]) for t in c.tensors[:2])
    assert k[66000, 0, 0, 0].item() == 66000 % 251 + 1000


# ------------------------------------------------------------------------------------------------------------- together
def test_offsets_beyond_32_bits():
    """The last sequence of a cache of more than 2^32 codes: written, read by both attention kernels, and moved."""
    seqs, nkv, context, dim, nq = 33, 4, 1 << 18, 128, 32
    assert seqs * nkv * context * dim > 1 << 32
    code = [torch.zeros(seqs, nkv, context, dim, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scale = [torch.zeros(seqs, nkv, context, device="cuda") for _ in range(2)]
    g = torch.Generator(device="cuda").manual_seed(3)
    for t, f in zip(code, scale):
        t[-1] = (60 * torch.randn(nkv, context, dim, device="cuda", generator=g)).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        f[-1] = 0.01 * torch.rand(nkv, context, device="cuda", generator=g)
    c = m.KvCache(code[0], code[1], scale[0], scale[1])
    host = lambda t, f, h, n: t[-1, h, :n].view(torch.float8_e4m3fn).double().cpu().numpy() * f[-1, h, :n].double().cpu().numpy()[:, None]  # noqa: E731
    work = torch.empty(m.tree_attention_workspace(dim), dtype=torch.uint8, device="cuda")
    for rows in (3, 40):
        prefix = context - rows
        slots = ints(range(prefix, context))
        qkv = torch.randn(rows, (nq + 2 * nkv) * dim, device="cuda", generator=g)
        q = torch.empty(rows, nq, dim, dtype=torch.bfloat16, device="cuda")
        out, status = torch.empty_like(q), ints([0])
        m.kv_write(c, m.Rope(dim, rotary_dim=0), qkv, nq, slots, q, seqs=ints([seqs - 1] * rows), slots=slots, status=status)
        m.tree_attention(c, q, ints([0, rows]), ints([prefix]), out, work, cache_seq=ints([seqs - 1]), status=status)
        torch.cuda.synchronize()
        assert status.item() == 0
        wrote = qkv.view(rows, -1, dim)[:, nq + nkv - 1].double().cpu().numpy()
        got = host(code[0], scale[0], nkv - 1, context)[prefix:]
        assert np.all(np.abs(got - wrote) <= H_E4M3 * np.abs(wrote) + 2.0 ** -10 * np.abs(wrote).max(1, keepdims=True) / 448 * 1.001)
        heads = slice(nq - nq // nkv, nq)
        for r in (0, rows - 1):
            want, tol = exact_attention(q[r, heads].double().cpu().numpy(), host(code[0], scale[0], nkv - 1, context),
                                        host(code[1], scale[1], nkv - 1, context), np.arange(context) <= prefix + r, dim ** -0.5)
            err = np.abs(out[r, heads].double().cpu().numpy() - want)
            assert np.all(err <= tol), (rows, r, float(err.max()))
    last = code[0][-1, :, context - 1].clone()
    m.kv_accept(m.KvCaches([c]), ints([context - 40]), ints([[39]]), ints([1]), cache_seq=ints([seqs - 1]))
    torch.cuda.synchronize()
    assert torch.equal(code[0][-1, :, context - 40], last) and not code[0][:-1].any()


def test_first_calls_inside_a_capture():
    """A process whose first calls are captured: nothing is set up that a capture forbids."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    script = """
import sys; sys.path.insert(0, %r)
import torch
from helpers import nfm
m = nfm()
g = torch.Generator(device="cuda").manual_seed(1)
k, v = (torch.randn(2, 2, 64, 128, device="cuda", generator=g).bfloat16() for _ in range(2))
qkv = torch.randn(40, 20 * 128, device="cuda", generator=g)
i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
slots, seqs, start, prefix = i(list(range(20)) * 2), i([0] * 20 + [1] * 20), i([0, 20, 40]), i([0, 0])
path, length, target = i([[1], [2]]), i([1, 1]), i([3] * 40)
q = torch.empty(40, 16, 128, dtype=torch.bfloat16, device="cuda")
out, lp = torch.zeros_like(q), torch.zeros(40, device="cuda")
work = torch.empty(m.tree_attention_workspace(128), dtype=torch.uint8, device="cuda")
c, rope = m.KvCache(k, v), m.Rope(128)
cs = m.KvCaches([c])
def step(s):
    m.kv_write(c, rope, qkv, 16, slots, q, seqs=seqs, slots=slots, stream=s)
    m.tree_attention(c, q, start, prefix, out, work, stream=s)                       # many rows
    m.tree_attention(c, q[:2], i2, prefix, out[:2], work, stream=s)                  # few
    m.token_logprobs(out.view(40, -1), target, lp, None, None, None, work, stream=s)
    m.kv_accept(cs, prefix, path, length, stream=s)
i2 = i([0, 1, 2])
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    step(torch.cuda.current_stream().cuda_stream)
k0, v0 = k.clone(), v.clone()
graph.replay(); torch.cuda.synchronize()
first = [t.clone() for t in (out, lp, k, v)]
k.copy_(k0); v.copy_(v0); step(0); torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(first, (out, lp, k, v)))
print("same")
""" % here
    r = subprocess.run([sys.executable, "-c", script], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("same"), r.stderr[-2000:]


@pytest.mark.parametrize("kind", ["e4m3", "bf16"])
def test_operators_in_a_graph_on_a_side_stream(kind):
    """Write, attend, log-probabilities and accept captured on another stream and replayed give what the eager calls give;
    two graphs that share a workspace, replayed in turn, each keep their results."""
    rng = np.random.default_rng(77)
    tokens, nq, nkv, dim = 6, 8, 1, 128
    x = torch.from_numpy(rng.standard_normal((tokens, (nq + 2 * nkv) * dim)).astype(np.float32)).cuda()
    start, prefix, seq, slot = ints([0, 4, 6]), ints([100, 7]), ints([0] * 4 + [1] * 2), ints([100, 101, 102, 103, 7, 8])
    bits = torch.tensor([[1], [3], [5], [13], [1], [3]], dtype=torch.int64, device="cuda")
    work = torch.empty(m.tree_attention_workspace(dim), dtype=torch.uint8, device="cuda")
    lwork = torch.empty(m.token_logprobs_workspace(tokens, nq * dim, 4), dtype=torch.uint8, device="cuda")
    rope, target = m.Rope(dim), ints(range(6))

    def make():
        c, _, _ = make_cache(np.random.default_rng(5), kind, 2, nkv, 200, dim)
        o = dict(q=torch.zeros(tokens, nq, dim, dtype=torch.bfloat16, device="cuda"), lp=torch.zeros(tokens, device="cuda"),
                 ti=torch.zeros(tokens, 4, dtype=torch.int32, device="cuda"), tl=torch.zeros(tokens, 4, device="cuda"))
        o["o"] = torch.zeros_like(o["q"])
        return c, m.KvCaches([c]), o

    def step(c, cs, o, stream):
        m.kv_write(c, rope, x, nq, slot, o["q"], seqs=seq, slots=slot, stream=stream)
        m.tree_attention(c, o["q"], start, prefix, o["o"], work, mask=bits, stream=stream)
        m.token_logprobs(o["o"].view(tokens, -1), target, o["lp"], None, o["ti"], o["tl"], lwork, stream=stream)
        m.kv_accept(cs, prefix, ints_path, ints_len, stream=stream)

    ints_path, ints_len = ints([[0, 2, 3], [1, -1, -1]]), ints([3, 1])
    eager = make()
    step(*eager, 0)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    sets, graphs = [make(), make()], []
    for st in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            step(*st, torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for st in sets:
        for name in ("q", "o", "lp", "ti", "tl"):
            assert torch.equal(st[2][name], eager[2][name]), name
        for a, b in zip(cache_host(st[0]), cache_host(eager[0])):
            assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
