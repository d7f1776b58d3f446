"""The decoder stack over several rows of a sequence (nf_stack_verify,
nf_stack_logprobs, nf_stack_accept) and with E4M3 caches, on the small stack
of test_gpu_stack.py.

Tolerances: those of test_gpu_stack.py against the CPU oracle (final hidden
state within 5e-2, cosine 0.9995; greedy tokens equal where the oracle's margin
exceeds 0.02).  Two ways through the same stack take the same arithmetic up to
the order of F32 sums (2^-24 each) and to where a sum falls on either side of a
BF16 rounding (2^-8 of one value among hundreds): they are held to the same."""
import numpy as np
import pytest

from helpers import REPO, assert_close, load_module, nfm, workload

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
m, wl = nfm(), workload()
so = load_module("nf_stack_oracle", REPO / "oracle" / "stack_oracle.py")
CFG = wl.STACK_CONFIGS["tiny"]


@pytest.fixture(scope="module")
def model():
    return wl.make_stack(CFG, seed=5)


def make_stack(model, max_batch, max_context, kv):
    c = model.cfg
    st = m.DecoderStack(vocab=c["vocab"], hidden=c["hidden"], layers=c["layers"], dense_layers=c["dense_layers"],
                        bf16_expert_layers=c["bf16_expert_layers"], dense_inter=c["dense_inter"],
                        experts=c["experts"], top_k=c["top_k"], inter=c["inter"], shared_inter=c["shared_inter"],
                        routed_scaling=c["scaling"], q_heads=c["q_heads"], kv_heads=c["kv_heads"],
                        max_batch=max_batch, max_context=max_context, kv=kv)
    st.bind_model(model)
    return st


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def e4m3_rows(x):
    """F32 rows [.., 128] as they read back from an E4M3 cache."""
    x = np.asarray(x, np.float32)
    scale = np.abs(x).max(-1, keepdims=True) * np.float32(1 / 448)
    code = torch.from_numpy((x / np.where(scale > 0, scale, 1)).astype(np.float32)).to(torch.float8_e4m3fn).float().numpy()
    return (code * scale).astype(np.float32)


def load_history(st, model, positions, max_batch, L, seed, kv):
    rng = np.random.default_rng(seed)
    nkv = model.cfg["kv_heads"]
    hist = [[], []]
    for l in range(len(model.layers)):
        bits = [wl.f32_to_bf16_bits(rng.standard_normal((max_batch, nkv, L, 128), dtype=np.float32)) for _ in range(2)]
        for b in bits:
            for i, p in enumerate(positions):
                b[i, :, p:] = 0
        st.load_kv(l, *bits)
        for h, b in zip(hist, bits):
            x = so.bf16_bits_to_f32(b).copy()
            h.append(e4m3_rows(x) if kv == "e4m3" else x)
    return hist


@pytest.fixture
def oracle_cache(monkeypatch):
    """The oracle's new cache rows (128 values) rounded as the cache's kind does."""
    def use(kv):
        if kv == "e4m3":
            plain = so.f32_to_bf16_f32
            monkeypatch.setattr(so, "f32_to_bf16_f32", lambda x: e4m3_rows(x) if np.shape(x) == (128,) else plain(x))
    return use


def check_rows(fin, nxt, want_next, logits, want_fin, what):
    assert_close(fin.cpu().numpy(), want_fin, max_abs=5e-2, min_cos=0.9995, what=what)
    srt = np.sort(logits, axis=1)
    clear = srt[:, -1] - srt[:, -2] > 0.02
    assert clear.sum() >= max(1, len(clear) // 2)
    assert np.array_equal(nxt.cpu().numpy()[clear], want_next[clear])


@pytest.mark.parametrize("kv", ["e4m3", "bf16"])
@pytest.mark.parametrize("batch", [3, 40])
def test_one_row_a_sequence_matches_the_oracle(model, oracle_cache, kv, batch):
    """nf_stack_verify with a row a sequence, and nf_stack_decode over E4M3 caches, are the oracle's step."""
    L = CFG["context"]
    rng = np.random.default_rng(batch)
    positions = rng.integers(0, L - 2, batch)
    positions[0], positions[-1] = 0, L - 2
    st = make_stack(model, batch, L, kv)
    k, v = load_history(st, model, positions, batch, L, batch, kv)
    oracle_cache(kv)
    tokens = rng.integers(0, CFG["vocab"], batch)
    nxt = torch.full((batch,), -1, dtype=torch.int32, device="cuda")
    fin = torch.empty((batch, CFG["hidden"]), dtype=torch.float32, device="cuda")
    st.verify(ints(tokens), ints(range(batch + 1)), ints(positions), batch, nxt, fin)
    st.sync()
    want = so.decode_step(model, k, v, tokens, positions)
    check_rows(fin, nxt, *want, "verify")
    if kv == "e4m3":
        tokens = want[0]
        st.decode(ints(tokens), ints(positions + 1), batch, nxt, fin)
        st.sync()
        check_rows(fin, nxt, *so.decode_step(model, k, v, tokens, positions + 1), "decode")
    st.close()


TREE = [-1, 0, 0, 1, 1, 2, 3, 5]  # parents of a tree of eight nodes


def tree_arrays(parents):
    bits, depth = [], []
    for i, p in enumerate(parents):
        bits.append((bits[p] if p >= 0 else 0) | 1 << i)
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return bits, depth


def path_to(parents, node):
    out = [node]
    while parents[out[0]] >= 0:
        out.insert(0, parents[out[0]])
    return out


def close(a, b, what):
    assert_close(a.cpu().numpy(), b.cpu().numpy(), max_abs=5e-2, min_cos=0.9995, what=what)


@pytest.mark.parametrize("kv", ["e4m3", "bf16"])
def test_a_tree_equals_its_paths_and_the_accepted_one_goes_on(model, kv):
    """Two sequences, one with a tree, one with a chain: every node's hidden state is that of its path alone (decoded token by
    token, and as a chain); after nf_stack_accept the next token goes on as behind the path."""
    H, V, L = CFG["hidden"], CFG["vocab"], CFG["context"]
    rng = np.random.default_rng(9)
    prefix = np.array([37, 5])
    bits, depth = tree_arrays(TREE)
    n = len(TREE)
    chain = 3
    tokens = rng.integers(0, V, n + chain)
    st = make_stack(model, 16, L, kv)

    def reset():
        load_history(st, model, prefix, 16, L, 77, kv)

    def verify(toks, starts, pre, **kw):
        rows = len(toks)
        fin = torch.empty((rows, H), dtype=torch.float32, device="cuda")
        nxt = torch.empty(rows, dtype=torch.int32, device="cuda")
        st.verify(ints(toks), ints(starts), ints(pre), rows, nxt, fin, **kw)
        st.sync()
        return fin, nxt

    reset()
    mask = torch.tensor([[b] for b in bits] + [[(1 << (i + 1)) - 1] for i in range(chain)], dtype=torch.int64, device="cuda")
    fin, nxt = verify(tokens, [0, n, n + chain], prefix, depth=ints(depth + list(range(chain))), mask=mask)

    # log-probabilities of the greedy tokens: the logits from the hidden states in 64 bits
    rows = n + chain
    lp, en = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    ti, tl = torch.empty(rows, 3, dtype=torch.int32, device="cuda"), torch.empty(rows, 3, device="cuda")
    st.logprobs(rows, nxt, lp, en, ti, tl)
    st.sync()
    logits = fin.double().cpu().numpy() @ so.bf16_bits_to_f32(model.lm_head).astype(np.float64).T
    full = logits - np.log(np.exp(logits - logits.max(1, keepdims=True)).sum(1, keepdims=True)) - logits.max(1, keepdims=True)
    tol = H * 2.0 ** -24 * (np.abs(fin.double().cpu().numpy()) @ np.abs(so.bf16_bits_to_f32(model.lm_head)).astype(np.float64).T).max() + 1e-5
    assert np.array_equal(ti[:, 0].cpu().numpy(), nxt.cpu().numpy())
    assert np.abs(lp.cpu().numpy() - full[np.arange(rows), nxt.cpu().numpy()]).max() <= 2 * tol
    assert torch.equal(lp, tl[:, 0]) and np.abs(en.cpu().numpy() + (np.exp(full) * full).sum(1)).max() <= 2 * tol * np.log(V)
    with pytest.raises(m.NfError, match="rows"):
        st.logprobs(rows + 1, None, None, en.repeat(2))

    path = path_to(TREE, 6)
    st.accept(ints(prefix), ints([path, [0, 1, 2, -1]]), ints([len(path), chain]))
    after, _ = verify([4, 7], [0, 1, 2], prefix + [len(path), chain])

    for leaf in (6, 4, 7):
        reset()
        p = path_to(TREE, leaf)
        got, _ = verify(list(tokens[p]) + list(tokens[n:]), [0, len(p), len(p) + chain], prefix)
        close(fin[p], got[:len(p)], f"path to {leaf} as a chain")
        close(fin[n:], got[len(p):], "the other sequence")
        reset()
        for j, node in enumerate(p):
            one, _ = verify([tokens[node], tokens[n + min(j, chain - 1)]], [0, 1, 2], [prefix[0] + j, prefix[1] + min(j, chain - 1)])
            close(fin[node:node + 1], one[:1], f"path to {leaf}, token {j}")
        if leaf == 6:
            go, _ = verify([4, 7], [0, 1, 2], prefix + [len(p), chain])
            close(after, go, "behind the accepted path")
    st.close()


@pytest.mark.parametrize("kv", ["e4m3", "bf16"])
def test_prompt_in_chunks_equals_token_by_token(model, kv):
    """A prompt of 21 tokens from an empty cache in chunks of 8, 12 and 1 rows ends as 21 single steps do."""
    L, H = CFG["context"], CFG["hidden"]
    rng = np.random.default_rng(3)
    prompt = rng.integers(0, CFG["vocab"], 21)
    st = make_stack(model, 16, L, kv)
    at = 0
    for n in (8, 12, 1):
        fin = torch.empty((n, H), dtype=torch.float32, device="cuda")
        st.verify(ints(prompt[at:at + n]), ints([0, n]), ints([at]), n, final_dev=fin)
        at += n
    st.sync()
    one = torch.empty((1, H), dtype=torch.float32, device="cuda")
    nxt = torch.empty(1, dtype=torch.int32, device="cuda")
    for i, t in enumerate(prompt):
        st.decode(ints([t]), ints([i]), 1, nxt, one)
    st.sync()
    close(fin[-1:], one, "the prompt's last token")
    st.close()


def test_verify_in_a_graph_and_padded_rows(model):
    """A captured step replayed with other tokens and prefixes in its buffers, rows behind the last sequence among them, is the
    eager step; the padding writes nothing to the caches."""
    L, H, B = 64, CFG["hidden"], 6
    st = make_stack(model, B, L, "e4m3")
    st.fill_kv(4)
    tok, start, pre = ints([1, 2, 3, 4, 0, 0]), ints([0, 3, 4]), ints([10, 20])
    fin = torch.zeros((B, H), dtype=torch.float32, device="cuda")
    nxt = torch.zeros(B, dtype=torch.int32, device="cuda")
    st.verify(tok, start, pre, B, nxt, fin)  # the first step sets attributes up
    st.sync()
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        st.verify(tok, start, pre, B, nxt, fin, stream=torch.cuda.current_stream().cuda_stream)
    st.fill_kv(4)
    tok.copy_(ints([9, 8, 7, 6, 5, 0]))
    start.copy_(ints([0, 1, 5]))
    pre.copy_(ints([30, 40]))
    g.replay()
    torch.cuda.synchronize()
    got, got_next = fin[:5].clone(), nxt[:5].clone()
    st.fill_kv(4)
    st.verify(tok, start, pre, 5, nxt[:5], fin[:5])
    st.sync()
    close(got, fin[:5], "replayed")
    assert torch.equal(got_next, nxt[:5])
    st.close()


def test_stack_refusals(model):
    st = make_stack(model, 4, 64, "e4m3")
    one = ints([1])
    nxt = torch.empty(1, dtype=torch.int32, device="cuda")
    with pytest.raises(m.NfError, match="not BF16"):
        st.kv_cache(0)
    d = st.kv_desc(1)
    assert (d.kind, d.seqs, d.kv_heads, d.max_context, d.head_dim) == (m.KV_E4M3, 4, CFG["kv_heads"], 64, 128) and d.k_scale
    for bad in (lambda: st.verify(ints(range(5)), ints([0, 5]), one, 5), lambda: st.verify(one, ints([0, 1]), one[:0], 1),
                lambda: st.verify(one, ints([0, 1]), one, 1, mask=torch.zeros(1, 65, dtype=torch.int64, device="cuda")),
                lambda: st.verify(one.long(), ints([0, 1]), one, 1), lambda: st.logprobs(1, None, None, None),
                lambda: st.accept(ints([0] * 5), ints([[0]] * 5), ints([1] * 5)), lambda: st.kv_desc(99),
                lambda: m.DecoderStack(vocab=10, hidden=256, layers=1, dense_layers=0, bf16_expert_layers=0, dense_inter=0, experts=4,
                                       top_k=1, inter=128, shared_inter=0, routed_scaling=1.0, q_heads=8, kv_heads=1, kv="int8")):
        with pytest.raises(m.NfError):
            bad()
    st.verify(one, ints([0, 1]), ints([63]), 1, nxt)  # the cache's last position
    st.sync()
    for prefix in (64, -1):
        st.verify(one, ints([0, 1]), ints([prefix]), 1, nxt)
        with pytest.raises(m.NfError, match="outside the cache"):
            st.sync()
    st.accept(ints([10]), ints([[3, 2]]), ints([2]))
    with pytest.raises(m.NfError, match="outside the cache"):
        st.sync()
    st.close()


def test_tp_logprobs():
    """A one-GPU group's log-probabilities read the last linear's output, whichever gather buffer holds it."""
    V, K, T = 700, 64, 5
    tp = m.TpGroup(8, V)
    g = torch.Generator().manual_seed(1)
    for step in range(3):
        w = torch.randn(V, K, generator=g).bfloat16().cuda()
        x = torch.randn(T, K, generator=g).cuda()
        tp.linear_bf16(w, V, K, x, T)
        target = torch.randint(0, V, (T,), generator=g).int().cuda()
        lp, en = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
        ti, tl = torch.empty(T, 4, dtype=torch.int32, device="cuda"), torch.empty(T, 4, device="cuda")
        tp.logprobs(T, V, target, lp, en, ti, tl)
        full = torch.log_softmax(x.double() @ w.double().T, -1)
        # the logits' F32 sums of K terms, twice
        tol = 2 * K * 2.0 ** -24 * float((x.double().abs() @ w.double().abs().T).max()) + 1e-5
        assert (lp.double() - full.gather(1, target.long()[:, None])[:, 0]).abs().max() <= tol
        assert (en.double() + (full.exp() * full).sum(-1)).abs().max() <= 10 * tol
        assert torch.equal(ti.long(), full.topk(4).indices) and (tl.double() - full.topk(4).values).abs().max() <= tol
    for bad in (lambda: tp.logprobs(9, V, None, None, en), lambda: tp.logprobs(T, V + 1, None, None, en),
                lambda: tp.logprobs(T, V, target, None, en), lambda: tp.logprobs(T, V, None, None, None, ti, None)):
        with pytest.raises(m.NfError):
            bad()
    tp.close()
