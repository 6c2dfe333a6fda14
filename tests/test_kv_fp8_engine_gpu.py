"""The e4m3 KV cache in use: the operators one after the other as a model calls them, and the engine
with an e4m3 cache, with and without a shared prefix."""
import pytest
import torch

from test_kv_fp8_gpu import D, PAGE, _check_status, _close, _empty_cache, _gen, _oracle, _tables, _values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv", [(8, 2), (32, 4), (4, 4)])
def test_write_prefill_write_decode(hq, hkv):
    """A layer's calls: three prompts on a shared prefix are written and attended, then three decode
    steps; every output against 64 bits over the values that the cache holds (read back)."""
    from swarm_inference_lab_b200.ops import attention, rope
    prefix, own = 128, [70, 1, 133]
    lens = [prefix + n for n in own]
    steps = 3
    table = _tables([n + steps for n in lens], 20, 1, shared=prefix // PAGE)
    k, v, sc = _empty_cache(20, hkv)
    cos_sin = rope.rope_cos_sin_table(512, D, 10000.0, device="cuda")
    g = _gen(hq)
    norm = (1 + 0.1 * torch.randn(D, device="cuda", generator=g)).bfloat16()

    def qkv(n):
        return torch.randn(n, (hq + 2 * hkv) * D, device="cuda", generator=g).bfloat16()

    def slots(seq, positions):
        return table[seq, positions // PAGE] * PAGE + positions % PAGE

    def write(x, seqs, positions):
        s = torch.cat([slots(i, p) for i, p in zip(seqs, positions)]).int()
        return rope.rope_kv_write_fp8(x, torch.cat(positions).int(), s, cos_sin, k, v, sc, hq, hkv, norm, norm)

    def span(a, b):
        return torch.arange(a, b, device="cuda")

    write(qkv(prefix), [0], [span(0, prefix)])                        # the prefix, once
    q = write(qkv(sum(own)), range(3), [span(prefix, n) for n in lens])
    cu = torch.tensor([0, 70, 71, 204], device="cuda", dtype=torch.int32)
    lens_t = torch.tensor(lens, device="cuda", dtype=torch.int32)
    out = attention.paged_prefill_fp8(q, k, v, sc, table, lens_t, cu, max(own))
    _check_status()
    _close(out, *_oracle(q, k, v, sc, table, lens, own))
    shared = torch.tensor([prefix], device="cuda", dtype=torch.int32)
    for _ in range(steps):
        q = write(qkv(3), range(3), [span(n, n + 1) for n in lens])
        lens = [n + 1 for n in lens]
        lens_t += 1
        want, tol = _oracle(q, k, v, sc, table, lens, [1, 1, 1])
        _close(attention.paged_decode_fp8(q, k, v, sc, table, lens_t), want, tol)
        _close(attention.paged_decode_shared_fp8(q, k, v, sc, table, lens_t, shared), want, tol)
        _check_status()
    # what the cache holds, read back, is what the oracle used
    at = slots(2, span(0, lens[2])).int()
    rk, rv = attention.read_kv_fp8(k, v, sc, at)
    page, off = at.long() // PAGE, at.long() % PAGE
    assert torch.equal(rk.double(), _values(k[page, :, off], sc[page, :, 0, off]))
    assert torch.equal(rv.double(), _values(v[page, :, off], sc[page, :, 1, off]))


def _engine(**kw):
    from swarm_inference_lab_b200.engine.engine import LLMEngine
    from swarm_inference_lab_b200.models.config import TINY_LLAMA_GPU
    from swarm_inference_lab_b200.models.dense import DenseWeights, TPInfo
    w = DenseWeights.random(TINY_LLAMA_GPU, TPInfo(), "cuda", seed=3, std=0.06)
    return LLMEngine(TINY_LLAMA_GPU, device="cuda", weights=w, max_batch=8, max_seq_len=512, kv_pages=64, **kw)


def _prompts(sizes, prefix=()):
    g = torch.Generator().manual_seed(4)
    return [list(prefix) + torch.randint(0, 4096, (n,), generator=g).tolist() for n in sizes]


def test_engine_with_an_e4m3_cache():
    """Same tokens from run to run and with and without graphs; all pages come back; and a cache of
    exactly the quantised rows."""
    from swarm_inference_lab_b200.engine.engine import SamplingParams
    prompts = _prompts([5, 70, 130])
    eng = _engine(kv_dtype="fp8")
    assert eng.kv.k.dtype == torch.float8_e4m3fn
    first = [o.token_ids for o in eng.generate(prompts, SamplingParams(max_new_tokens=12))[0]]
    again = [o.token_ids for o in eng.generate(prompts, SamplingParams(max_new_tokens=12))[0]]
    eager = _engine(kv_dtype="fp8", use_cuda_graphs=False)
    third = [o.token_ids for o in eager.generate(prompts, SamplingParams(max_new_tokens=12))[0]]
    _check_status()
    assert first == again == third and all(len(t) == 12 for t in first)
    assert eng.kv.alloc.free == 64 and not eng.kv.seqs
    sampled = [o.token_ids for o in eng.generate(prompts, SamplingParams(max_new_tokens=6, temperature=0.8, seed=5))[0]]
    _check_status()
    assert all(len(t) == 6 for t in sampled)


@pytest.mark.parametrize("decode", [False, True])
def test_hidden_states_differ_from_a_bf16_cache_by_the_quantisation(decode):
    """Two layers with an e4m3 cache beside the same with a bf16 one.  A code is within 2^-4 of its
    value, so a score moves by at most 2^-4 sum|q k| and a value by 2^-4 of itself: the attention
    output by some 2^-3 of its size at worst, which the residual stream (that keeps the embedding and
    the MLPs) halves; two layers of that stay under 2^-2 of the stream's norm."""
    from swarm_inference_lab_b200.engine.kv_cache import PagedKVCache
    from swarm_inference_lab_b200.models.config import TINY_LLAMA_GPU as cfg
    from swarm_inference_lab_b200.models.dense import DenseModel, DenseWeights, ForwardBatch, TPInfo
    model = DenseModel(DenseWeights.random(cfg, TPInfo(), "cuda", seed=5), "cuda", max_positions=1024)
    T = 100
    ids = torch.randint(0, cfg.vocab_size, (T + 1,), device="cuda", generator=_gen(1))

    def batch(a, b, is_decode):
        n = b - a
        return ForwardBatch(ids=ids[a:b], positions=torch.arange(a, b, dtype=torch.int32, device="cuda"),
                            slots=torch.arange(a, b, dtype=torch.int32, device="cuda"),
                            seq_lens=torch.tensor([b], dtype=torch.int32, device="cuda"),
                            block_table=torch.arange(16, dtype=torch.int32, device="cuda")[None],
                            last_idx=torch.arange(n, device="cuda"), is_decode=is_decode,
                            cu_q=torch.tensor([0, n], dtype=torch.int32, device="cuda"), max_q_len=n)

    out = {}
    for kind in ("bf16", "fp8"):
        kv = PagedKVCache(cfg.num_layers, cfg.num_kv_heads, 16, "cuda", kv_dtype=kind)
        out[kind] = model.forward_hidden(batch(0, T, False), kv).float()
        if decode:
            out[kind] = model.forward_hidden(batch(T, T + 1, True), kv).float()
    _check_status()
    diff = (out["fp8"] - out["bf16"]).norm() / out["bf16"].norm()
    assert 0 < diff < 0.25, diff.item()


@pytest.mark.parametrize("kv_dtype", ["fp8", "bf16"])
def test_shared_prefix_in_the_engine(kv_dtype):
    """Requests on a shared prefix: its pages are written once, every request gets all its tokens, the
    pages come back, and a request that does not share (or is the prefix alone) is served as before."""
    from swarm_inference_lab_b200.engine.engine import SamplingParams
    prefix = _prompts([200])[0]
    eng = _engine(kv_dtype=kv_dtype)
    assert eng.set_shared_prefix(prefix) == 192
    assert eng.kv.alloc.free == 64 - 3
    prompts = _prompts([9, 1, 70, 33], prefix[:192])
    outs, _ = eng.generate(prompts, SamplingParams(max_new_tokens=10))
    _check_status()
    assert [len(o.token_ids) for o in outs] == [10] * 4
    assert eng.kv.alloc.free == 64 - 3 and eng.kv.alloc.refcount(eng.kv.seqs["\0shared prefix"].pages[0]) == 1
    if kv_dtype == "fp8":
        assert any(shared for _, _, shared in eng.runner.graphs)
    again, _ = eng.generate(prompts, SamplingParams(max_new_tokens=10))
    assert [o.token_ids for o in again] == [o.token_ids for o in outs]
    # a batch with a request that does not share, and one that is no longer than the prefix
    mixed = [prompts[0], _prompts([20])[0], prefix[:192]]
    outs2, _ = eng.generate(mixed, SamplingParams(max_new_tokens=5))
    _check_status()
    plain = _engine(kv_dtype=kv_dtype)
    alone, _ = plain.generate(mixed[1:], SamplingParams(max_new_tokens=5))
    assert [len(o.token_ids) for o in outs2] == [5] * 3 and len(alone) == 2
    rid = eng.add_request(prompts[0])
    with pytest.raises(ValueError, match="no request"):
        eng.set_shared_prefix([])
    eng.cancel(rid)
    assert eng.set_shared_prefix([]) == 0
    assert eng.kv.alloc.free == 64 and not eng.kv.seqs
    with pytest.raises(ValueError, match="no room"):
        eng.set_shared_prefix(list(range(512)))


def test_rows_of_a_sequence():
    """The rows that a sequence holds, from either kind of cache, are the ones that were written."""
    from swarm_inference_lab_b200.engine.kv_cache import PagedKVCache
    from swarm_inference_lab_b200.ops import rope
    hkv, T = 2, 100
    qkv = torch.randn(T, 6 * D, device="cuda", generator=_gen(2)).bfloat16()
    cos_sin = rope.rope_cos_sin_table(128, D, 10000.0, device="cuda")
    got = {}
    for kind in ("bf16", "fp8"):
        kv = PagedKVCache(1, hkv, 4, "cuda", kv_dtype=kind)
        kv.open("x")
        kv.reserve("x", T)
        slots = torch.tensor(kv.slots("x", 0, T), dtype=torch.int32, device="cuda")
        pos = torch.arange(T, dtype=torch.int32, device="cuda")
        if kind == "fp8":
            rope.rope_kv_write_fp8(qkv.clone(), pos, slots, cos_sin, *kv.layer(0), kv.layer_scales(0), 2, hkv)
        else:
            rope.rope_kv_write(qkv.clone(), pos, slots, cos_sin, *kv.layer(0), 2, hkv)
        got[kind] = kv.rows(0, "x", 30, 65)
    _check_status()
    assert torch.equal(got["bf16"][1], qkv.unflatten(1, (6, D))[30:95, 4:])
    for a, b in zip(got["fp8"], got["bf16"]):
        a, b = a.double(), b.double()
        # e4m3: half a step of a value, or of the smallest one that the scale (at most 2 max / 448) has;
        # the bf16 rows are rounded themselves
        amax = b.abs().amax(-1, keepdim=True)
        assert ((a - b).abs() <= 2.0 ** -4 * b.abs() + 2.0 ** -10 * 2 * amax / 448 + 2.0 ** -8 * amax).all()


def _tiny(moe=False, **kw):
    from swarm_inference_lab_b200.engine.engine import LLMEngine
    from swarm_inference_lab_b200.models.config import TINY_LLAMA_GPU, ModelConfig
    from swarm_inference_lab_b200.models.dense import DenseWeights, TPInfo
    from swarm_inference_lab_b200.models.moe import MoEWeights
    cfg, weights = TINY_LLAMA_GPU, DenseWeights
    if moe:
        cfg, weights = ModelConfig(name="tiny-moe", family="qwen3_moe", vocab_size=2048, hidden_size=512, num_layers=2,
                                   num_heads=4, num_kv_heads=2, head_dim=128, intermediate_size=1024, qk_norm=True,
                                   num_experts=8, num_experts_per_tok=2, moe_intermediate_size=256,
                                   rms_norm_eps=1e-6), MoEWeights
    return LLMEngine(cfg, device="cuda", weights=weights.random(cfg, TPInfo(), "cuda", seed=3, std=0.06), **kw)


def test_a_prefix_over_half_the_cache_serves_requests_together():
    """The prefix's pages are there once: a request on them needs its own pages only."""
    from swarm_inference_lab_b200.engine.engine import SamplingParams
    eng = _tiny(max_batch=8, max_seq_len=3000, kv_pages=64, kv_dtype="fp8")
    prefix = _prompts([40 * PAGE])[0]
    assert eng.set_shared_prefix(prefix) == 40 * PAGE
    prompts = [prefix + t for t in _prompts([10, 60, 1, 100, 5, 6, 7, 8])]
    for p in prompts:
        eng.add_request(p, SamplingParams(max_new_tokens=5))
    assert len(eng.step()) == 8                                # all of them are admitted at once
    assert eng.kv.alloc.free == 24 - 10                        # (two need two pages)
    with pytest.raises(ValueError, match="KV tokens"):         # one that does not share has 24 pages
        eng.add_request(_prompts([24 * PAGE])[0], SamplingParams(max_new_tokens=1))
    while eng.scheduler.has_work():
        eng.step()
    _check_status()
    assert eng.kv.alloc.free == 24


def test_a_shared_prefix_that_cannot_be_set_leaves_the_engine_without_one():
    from swarm_inference_lab_b200.engine.engine import SamplingParams
    from swarm_inference_lab_b200.engine.kv_cache import OutOfPages
    eng = _tiny(max_batch=8, max_seq_len=512, kv_pages=64, kv_dtype="fp8")
    prefix = _prompts([200])[0]
    prefill = eng.runner.prefill

    def broken(*a, **kw):
        raise RuntimeError("prefill failed")

    for how in ("pages", "prefill"):
        assert eng.set_shared_prefix(prefix) == 192
        if how == "pages":
            eng.kv.open("x")
            eng.kv.reserve("x", 61 * PAGE)
            with pytest.raises(OutOfPages):
                eng.set_shared_prefix(prefix + prefix)
            eng.kv.close("x")
        else:
            eng.runner.prefill = broken
            with pytest.raises(RuntimeError, match="prefill failed"):
                eng.set_shared_prefix(prefix)
            eng.runner.prefill = prefill
        assert eng.kv.alloc.free == 64 and not eng.kv.seqs
        assert eng.scheduler.kv_capacity == 64 * PAGE and int(eng.runner.prefix_len) == 0
        out, _ = eng.generate([prefix + [1]], SamplingParams(max_new_tokens=3))
        assert len(out[0].token_ids) == 3 and eng.kv.alloc.free == 64
    _check_status()


def _served(eng, prompt, n):
    """Tokens of one request served alone, and the logits that each was taken from."""
    from swarm_inference_lab_b200.engine.engine import SamplingParams
    logits, seen = eng.model.logits, []

    def keep(h, fb):
        seen.append(logits(h, fb))
        return seen[-1]

    eng.model.logits = keep
    try:
        out = eng.generate([prompt], SamplingParams(max_new_tokens=n))[0][0].token_ids
    finally:
        eng.model.logits = logits
    return out, [x[:1].clone() for x in seen[-n:]]


@pytest.mark.parametrize("kv_dtype", ["fp8", "bf16"])
def test_requests_on_a_shared_prefix_are_those_of_an_engine_without_one(kv_dtype):
    """An engine whose prefill budget is the prefix's length computes a prompt's first 192 tokens in one
    call, as the engine with a shared prefix did beforehand, and the rest in another: every shape is the
    same, so tokens and logits must be, bit for bit.  A second prefix of another length, a request that
    does not share, and one that is the prefix alone go through the same engine."""
    kw = dict(max_batch=8, max_seq_len=512, kv_pages=64, kv_dtype=kv_dtype, use_cuda_graphs=False)
    first, second = _prompts([200])[0], _prompts([320, 330])[1]
    sharing = _tiny(prefill_token_budget=320, **kw)
    for prefix, n in ((first, 192), (second, 320)):
        plain = _tiny(prefill_token_budget=n, **kw)
        assert sharing.set_shared_prefix(prefix) == n
        seen = []
        for tail in (1, 70, 33):
            prompt = prefix[:n] + _prompts([tail])[0]
            (a, la), (b, lb) = _served(sharing, prompt, 4), _served(plain, prompt, 4)
            assert a == b and len(la) == 4 and all(torch.equal(x, y) for x, y in zip(la, lb))
            seen += la
        for prompt in (_prompts([20])[0], prefix[:n]):
            (a, la), (b, lb) = _served(sharing, prompt, 4), _served(plain, prompt, 4)
            assert a == b and all(torch.equal(x, y) for x, y in zip(la, lb))
        assert not any(torch.equal(x, y) for x, y in zip(seen, seen[4:]))
    _check_status()


def test_a_decode_batch_on_a_prefix_that_is_attended_apart():
    """The hidden states of a decode step through the shared-prefix operator against those of the same
    step row by row: both attend to the same rows and round each attention output to bf16, so they differ
    by roundings, and another prefix (whose hidden states are computed for comparison) changes them by the
    size of the attention itself.  An eighth of that change is far above the roundings (2^-8 per output
    and layer) and far below any row or page read wrongly.  With graphs the tokens are the same, also
    after the prefix was replaced by one of another length."""
    from swarm_inference_lab_b200.engine.engine import SamplingParams
    kw = dict(max_batch=64, max_seq_len=4160, kv_pages=1600, kv_dtype="fp8")
    eager, graphs = _tiny(use_cuda_graphs=False, **kw), _tiny(**kw)
    assert 64 * 2 * eager.runner.max_pages > 8192              # (attended apart from here on)
    texts = _prompts([1100, 1500, 1500])
    tails = _prompts([3 + i % 7 for i in range(50)])
    for text, other in ((texts[0], texts[1]), (texts[1], texts[2])):
        n = eager.set_shared_prefix(text)
        assert n == len(text) // PAGE * PAGE == graphs.set_shared_prefix(text)
        rids = [eager.add_request(text[:n] + t, SamplingParams(max_new_tokens=4)) for t in tails]
        eager.step()
        reqs = [eager.scheduler.running[r] for r in rids]
        ids, at = [r.output[-1] for r in reqs], [r.context_len - 1 for r in reqs]
        pages = [list(eager.kv.seqs[r].pages) for r in rids]

        def hidden(pages, shared):
            dg = eager.runner.graph_for(64, shared=shared)
            eager.runner.stage_decode_inputs(dg, ids, at, pages)
            return eager.model.forward_hidden(dg.fb, eager.kv)[:50].float()

        together, alone = hidden(pages, True), hidden(pages, False)
        _check_status()
        eager.kv.open("other")
        instead = eager.kv.reserve("other", n).pages
        eager.runner.prefill([other[:n]], [0], [instead])
        changed = hidden([instead + p[n // PAGE:] for p in pages], False)
        eager.kv.close("other")
        change = (changed - alone).norm(dim=1)
        assert ((together - alone).norm(dim=1) < change / 8).all()
        for r in rids:
            eager.cancel(r)
        outs = [[o.token_ids for o in e.generate([text[:n] + t for t in tails], SamplingParams(max_new_tokens=4))[0]]
                for e in (eager, graphs)]
        _check_status()
        assert outs[0] == outs[1] and any(shared for _, _, shared in graphs.runner.graphs)


@pytest.mark.parametrize("moe", [False, True])
def test_sampled_requests_on_a_shared_prefix(moe):
    """Drawn tokens are the same from run to run, with and without graphs, in a dense and a mixture model."""
    from swarm_inference_lab_b200.engine.engine import SamplingParams
    kw = dict(moe=moe, max_batch=8, max_seq_len=512, kv_pages=64, kv_dtype="fp8")
    prefix = torch.randint(0, 2048, (200,), generator=torch.Generator().manual_seed(1)).tolist()
    prompts = [prefix[:192] + [i, 7, 9][:1 + i % 3] for i in range(4)]
    params = SamplingParams(max_new_tokens=6, temperature=0.8, top_k=50, repetition_penalty=1.1, seed=5)
    got = []
    for graphs in (True, True, False):
        eng = _tiny(use_cuda_graphs=graphs, **kw)
        assert eng.set_shared_prefix(prefix) == 192
        got.append([o.token_ids for o in eng.generate(prompts, params)[0]])
        _check_status()
        assert any(shared and sampled for _, sampled, shared in eng.runner.graphs)
    assert got[0] == got[1] == got[2] and all(len(t) == 6 for t in got[0])
