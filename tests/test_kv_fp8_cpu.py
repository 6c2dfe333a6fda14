"""The e4m3 KV cache's format on the CPU: quantisation against a search over all codes, and calls
that are refused without a GPU."""
import math

import pytest
import torch

from swarm_inference_lab_b200.ops import kv_fp8


def _codes():
    """Every finite e4m3 value with its code, from the format's definition."""
    out = {}
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        if e == 15 and m == 7:
            continue
        mag = m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        out[c] = -mag if c & 128 else mag
    return out


def test_e4m3_bytes_are_the_formats():
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    for c, x in _codes().items():
        assert t[c].item() == x


@pytest.mark.parametrize("size", [1e-38, 1e-12, 1e-3, 1.0, 300.0, 1e6, 1e20, 3e38])
def test_quantisation_is_the_nearest_code_of_the_smallest_scale(size):
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(6, 128, generator=g) * size).clamp(-3.3e38, 3.3e38)
    x[1] = x[1].bfloat16().float()
    x[2, 0] = 448.0 * 2.0 ** math.floor(math.log2(size) + 2) if size < 1e36 else x[2, 0]
    codes, scales = kv_fp8.kv_quantize_reference(x)
    values = _codes()
    table = torch.tensor(sorted(set(values.values())), dtype=torch.float64)
    for r in range(6):
        amax = x[r].abs().max().item()
        e = scales[r].item() - 127
        fits = [n for n in range(-60, 61) if amax <= 448.0 * 2.0 ** n]
        assert e == (fits[0] if fits else 60)
        y = (x[r].double() / 2.0 ** e).clamp(-448, 448)
        d = (y[:, None] - table[None]).abs()
        got = (kv_fp8.kv_dequantize_reference(codes[r], scales[r]).double() / 2.0 ** e)
        assert torch.equal((y - got).abs(), d.min(-1).values)
        tie = (d == d.min(-1, keepdim=True).values).sum(-1) > 1
        assert ((codes[r].view(torch.uint8) & 1)[tie] == 0).all()       # to the even code


def test_zero_and_non_finite_tokens():
    x = torch.ones(4, 128)
    x[0] = 0
    x[1, 7] = math.inf
    x[2, 9] = math.nan
    codes, scales = kv_fp8.kv_quantize_reference(x)
    assert scales.tolist() == [67, 255, 255, 127 - 8]
    y = kv_fp8.kv_dequantize_reference(codes, scales)
    assert (y[0] == 0).all() and torch.isnan(y[1]).all() and torch.isnan(y[2]).all() and (y[3] == 1).all()


def test_kernels_refuse_cpu_tensors():
    from swarm_inference_lab_b200.ops._ext import available, ext
    if not available():
        pytest.skip("kernel library not built")
    k = torch.zeros(2, 1, 64, 128).to(torch.float8_e4m3fn)
    sc = torch.zeros(2, 1, 2, 64, dtype=torch.uint8)
    i = torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 3 * 128, dtype=torch.bfloat16)
    status = torch.zeros(4, dtype=torch.int32)
    out = torch.zeros(1, 1, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="qkv must be bf16"):
        ext().rope_kv_write_fp8(x, i, i, torch.zeros(4, 128), None, None, 1e-6, k, k, sc, 1, 1, None, status)
    with pytest.raises(RuntimeError, match="KV cache"):
        ext().read_kv_fp8(k, k, sc, i, out, out, status)
    with pytest.raises(RuntimeError, match="KV cache"):
        ext().paged_decode_fp8(out, k, k, sc, torch.zeros(1, 1, dtype=torch.int32), i, x[:, :128], 0.1, status)


# ------------------------------------------------------------------ the cache object
def test_cache_pages_and_bytes():
    from swarm_inference_lab_b200.engine.kv_cache import PagedKVCache
    kv = PagedKVCache(2, 3, 8, "cpu", kv_dtype="fp8")
    assert kv.k.dtype == kv.v.dtype == torch.float8_e4m3fn and kv.k.shape == (2, 8, 3, 64, 128)
    assert kv.scales.shape == (2, 8, 3, 2, 64) and kv.layer_scales(1).data_ptr() == kv.scales[1].data_ptr()
    held = kv.k.numel() + kv.v.numel() + kv.scales.numel()
    assert PagedKVCache.bytes_per_page(2, 3, kv_dtype="fp8") * 8 == held
    plain = PagedKVCache(2, 3, 8, "cpu")
    assert plain.layer_scales(0) is None and plain.kv_dtype == "bf16" and plain.k.dtype == torch.bfloat16
    for kw in ({"kv_dtype": "e4m3"}, {"kv_dtype": "fp8", "latent_dim": 576}, {"kv_dtype": "fp8", "head_dim": 64}):
        with pytest.raises(ValueError):
            PagedKVCache(1, 1, 2, "cpu", **kw)


@pytest.mark.parametrize("kv_dtype", ["bf16", "fp8"])
def test_snapshot_and_restore(kv_dtype):
    from swarm_inference_lab_b200.engine.kv_cache import PagedKVCache
    g = torch.Generator().manual_seed(0)
    a, b = (PagedKVCache(2, 2, 6, "cpu", kv_dtype=kv_dtype) for _ in range(2))
    raw = (lambda t: t.view(torch.uint8)) if kv_dtype == "fp8" else (lambda t: t.view(torch.int16))
    for t in (a.k, a.v):
        raw(t).copy_(torch.randint(0, 100, raw(t).shape, generator=g))
    if a.scales is not None:
        a.scales.copy_(torch.randint(100, 150, a.scales.shape, generator=g))
    a.open("x"), b.open("other")
    b.reserve("other", 70)
    a.reserve("x", 130)
    a.seqs["x"].length = 130
    snap = a.snapshot("x")
    b.restore("x", snap)
    assert b.seqs["x"].length == 130 and b.seqs["x"].pages != a.seqs["x"].pages
    for i, j in zip(a.seqs["x"].pages, b.seqs["x"].pages):
        assert torch.equal(raw(a.k)[:, i], raw(b.k)[:, j]) and torch.equal(raw(a.v)[:, i], raw(b.v)[:, j])
        if a.scales is not None:
            assert torch.equal(a.scales[:, i], b.scales[:, j])
    other = PagedKVCache(2, 2, 6, "cpu", kv_dtype="bf16" if kv_dtype == "fp8" else "fp8")
    with pytest.raises(ValueError, match="snapshot"):
        other.restore("x", snap)
    assert "x" not in other.seqs and other.alloc.free == 6


def test_fork_prefix_shares_whole_pages_only():
    from swarm_inference_lab_b200.engine.kv_cache import PagedKVCache
    kv = PagedKVCache(1, 1, 10, "cpu", kv_dtype="fp8")
    kv.open("p")
    kv.reserve("p", 200)
    kv.seqs["p"].length = 200
    for n, pages in ((0, 0), (63, 0), (64, 1), (130, 2), (200, 3)):
        s = kv.fork_prefix("p", "q", n)
        assert s.pages == kv.seqs["p"].pages[:pages] and s.length == 64 * pages
        kv.reserve("q", 64 * pages + 1)
        assert s.pages[pages] not in kv.seqs["p"].pages          # its own page to write to
        kv.close("q")
        assert kv.alloc.free == 6
    for bad in (-1, 201):
        with pytest.raises(ValueError):
            kv.fork_prefix("p", "q", bad)
    kv.fork_prefix("p", "q", 64)
    with pytest.raises(KeyError):
        kv.fork_prefix("p", "q", 64)
    kv.close("p")
    assert kv.alloc.free == 9                                    # the shared page lives on
    kv.close("q")
    assert kv.alloc.free == 10


def test_rows_refusals():
    from swarm_inference_lab_b200.engine.kv_cache import PagedKVCache
    kv = PagedKVCache(1, 1, 4, "cpu")
    kv.open("x")
    kv.reserve("x", 100)
    k, v = kv.rows(0, "x", 60, 10)
    assert k.shape == v.shape == (10, 1, 128)
    for start, count in ((-1, 2), (120, 9), (0, -1)):
        with pytest.raises(ValueError):
            kv.rows(0, "x", start, count)
    with pytest.raises(ValueError):
        PagedKVCache(1, 1, 4, "cpu", latent_dim=576).rows(0, "x", 0, 1)


def test_a_shared_request_enters_the_scheduler_past_its_prefix():
    from swarm_inference_lab_b200.engine.scheduler import ContinuousScheduler, SeqRequest
    sch = ContinuousScheduler(max_batch=4, prefill_token_budget=100, kv_capacity_tokens=4096)
    sch.admit(SeqRequest("a", list(range(200)), 5, 0, prompt_consumed=128))
    it = sch.next_iteration()
    assert it.prefill == (("a", 72),)
    sch.mark_prefill("a", 72, 7)
    r = sch.running["a"]
    assert r.prefill_complete and r.context_len == 201 and r.output == [7]


def test_engine_refuses_other_cache_types():
    from swarm_inference_lab_b200.engine.engine import LLMEngine
    from swarm_inference_lab_b200.models.config import TINY_LLAMA_GPU, TINY_MLA_GPU
    with pytest.raises(ValueError, match="kv_dtype"):
        LLMEngine(TINY_LLAMA_GPU, device="cuda:0", kv_dtype="int8")
    with pytest.raises(ValueError, match="MLA"):
        LLMEngine(TINY_MLA_GPU, device="cuda:0", kv_dtype="fp8")


def test_cli_refuses_other_cache_types():
    from typer.testing import CliRunner
    from swarm_inference_lab_b200.cli import app
    r = CliRunner().invoke(app, ["run", "tiny-llama-gpu", "--kv-dtype", "int8"])
    assert r.exit_code != 0 and "kv-dtype" in r.output + str(r.exception)


def test_a_request_on_a_shared_prefix_is_charged_its_own_pages():
    """2560 shared tokens of 4096 and 1536 of room: requests of 2560 + 10 tokens need one page each."""
    from swarm_inference_lab_b200.engine.scheduler import ContinuousScheduler, SeqRequest
    sch = ContinuousScheduler(max_batch=64, prefill_token_budget=8192, kv_capacity_tokens=4096 - 2560)
    for i in range(30):
        sch.admit(SeqRequest(f"r{i}", list(range(2570)), 5, i, prompt_consumed=2560, shared_tokens=2560))
    it = sch.next_iteration()
    assert [n for _, n in it.prefill] == [10] * 24 and len(sch.waiting) == 6       # 24 pages are free
    assert sch.reserved_tokens == 24 * 64
    for rid, n in it.prefill:
        sch.mark_prefill(rid, n, 1)
    assert sch.reserved_tokens == 24 * 64                                          # not less as the prompt is taken in
    with pytest.raises(ValueError, match="KV tokens"):
        sch.admit(SeqRequest("own", list(range(2570)), 5, 99))
    with pytest.raises(ValueError, match="shared"):
        sch.admit(SeqRequest("odd", list(range(200)), 5, 99, shared_tokens=100))
    with pytest.raises(ValueError, match="shared"):
        sch.admit(SeqRequest("all", list(range(128)), 5, 99, shared_tokens=192))


@pytest.mark.parametrize("kv_dtype", ["bf16", "fp8"])
def test_truncating_a_fork_into_a_shared_page_copies_it(kv_dtype):
    """A sequence that is rolled back below the end of a page that it shares writes the page's rest again:
    into a copy of its own."""
    from swarm_inference_lab_b200.engine.kv_cache import OutOfPages, PagedKVCache
    kv = PagedKVCache(2, 2, 5, "cpu", kv_dtype=kv_dtype)
    raw = (lambda t: t.view(torch.uint8)) if kv_dtype == "fp8" else (lambda t: t.view(torch.int16))
    for t in (kv.k, kv.v):
        raw(t).copy_(torch.randint(0, 100, raw(t).shape, generator=torch.Generator().manual_seed(1)))
    if kv.scales is not None:
        kv.scales.copy_(torch.randint(100, 150, kv.scales.shape, generator=torch.Generator().manual_seed(2)))
    kv.open("p")
    kv.reserve("p", 128)
    kv.seqs["p"].length = 128
    old = list(kv.seqs["p"].pages)
    q = kv.fork_prefix("p", "q", 128)
    kv.truncate("q", 128)
    assert q.pages == old                                                          # nothing to write to
    kv.truncate("q", 70)
    assert q.length == 70 and q.pages[0] == old[0] and q.pages[1] not in old
    for t in (raw(kv.k), raw(kv.v)) + ((kv.scales,) if kv.scales is not None else ()):
        assert torch.equal(t[:, q.pages[1]], t[:, old[1]])
    assert kv.alloc.refcount(old[0]) == 2 and kv.alloc.refcount(old[1]) == 1 and kv.alloc.free == 2
    copy = q.pages[1]
    kv.truncate("q", 65)
    assert q.pages == [old[0], copy]                                               # its own by now
    kv.truncate("q", 64)
    assert q.pages == [old[0]] and kv.alloc.free == 3
    kv.open("z")
    kv.reserve("z", 192)
    with pytest.raises(OutOfPages):
        kv.truncate("q", 30)                                                       # no page for the copy
    assert q.pages == [old[0]] and q.length == 64 and kv.alloc.refcount(old[0]) == 2
    kv.close("z")
    kv.truncate("q", 0)
    assert q.pages == [] and q.length == 0 and kv.seqs["p"].pages == old
    kv.close("p"), kv.close("q")
    assert kv.alloc.free == 5


def test_cli_refuses_an_e4m3_cache_for_a_model_of_latent_rows():
    from typer.testing import CliRunner
    from swarm_inference_lab_b200.cli import app
    for args in ([], ["--dry-run"]):
        r = CliRunner().invoke(app, ["run", "tiny-mla-gpu", "--kv-dtype", "fp8", "--prompt", "x", *args])
        assert r.exit_code == 2 and "kv-dtype" in r.output, (r.exit_code, r.output, r.exception)
