"""Prompt attention against the formula in 64 bits."""
import pytest
import torch

from tests.ops_ref import HALF, attend, attend_fast, attention_bound, logit_error

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SC = 128 ** -0.5


@pytest.fixture(scope="module")
def kb():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import kitty_b200

    return kitty_b200


def _inputs(shape_q, shape_k, dtype, seed, qscale=0.7):
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = (qscale * torch.randn(shape_q, generator=g, device=DEV)).to(dtype)
    k = torch.randn(shape_k, generator=g, device=DEV)
    k[..., :4] *= 8.0
    v = torch.randn(shape_k, generator=g, device=DEV)
    return q, k.to(dtype), v.to(dtype)


def _limits(n, m, causal):
    i = torch.arange(n, device=DEV)
    return (i + 1 + m - n).clamp(0, m) if causal else torch.full((n,), m, device=DEV)


def _check_rows(got, q, k, v, scaling, causal, what=""):
    """got [n, H_Q, D], q [n, H_Q, D], k / v [m, H, D] of one sequence."""
    n, hq, _ = q.shape
    m, h, _ = k.shape
    lim = _limits(n, m, causal)
    for x in range(hq):
        qx, kx, vx = q[:, x].double(), k[:, x // (hq // h)].double(), v[:, x // (hq // h)].double()
        want, mag = attend_fast(qx, kx, vx, scaling, lim)
        bound = attention_bound(want, mag, q.dtype, HALF[q.dtype], logit_error(qx, kx, scaling))
        off = (got[:, x].double() - want).abs()
        assert (off <= bound).all(), (what, x, off.max().item(), (off - bound).max().item())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,hq,h,Lq,Lk", [
    (1, 1, 1, 1, 1), (1, 4, 1, 128, 128), (2, 8, 2, 127, 127), (1, 7, 1, 129, 129), (1, 28, 4, 300, 300),
    (2, 4, 4, 257, 257), (1, 8, 1, 640, 640), (1, 3, 1, 1, 777), (2, 4, 2, 100, 900), (1, 2, 2, 5, 133),
    (1, 32, 1, 70, 70), (1, 2, 1, 200, 90), (1, 1, 1, 1300, 1300)])
@pytest.mark.parametrize("causal", [True, False])
def test_dense(kb, dtype, B, hq, h, Lq, Lk, causal):
    q, k, v = _inputs((B, hq, Lq, 128), (B, h, Lk, 128), dtype, Lq + Lk)
    got = kb.prompt_attention(q, k, v, SC, causal=causal)
    assert got.shape == (B, Lq, hq, 128) and got.dtype == dtype
    for b in range(B):
        _check_rows(got[b], *(x[b].transpose(0, 1) for x in (q, k, v)), SC, causal)
    # projection layout, read in place
    qt, kt, vt = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v))
    assert torch.equal(kb.prompt_attention(qt, kt, vt, SC, causal=causal), got)
    assert kb.prompt_attention_status(DEV) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,h", [(28, 4), (4, 4), (3, 1)])
@pytest.mark.parametrize("lens", [[1, 37, 128, 129, 300], [0, 5, 0, 0, 513, 1, 256], [700], [0], [1] * 70])
def test_packed(kb, dtype, hq, h, lens):
    T = sum(lens)
    extra = 3
    q, k, v = _inputs((T + extra, hq, 128), (T + extra, h, 128), dtype, T)
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
    k[T:], v[T:] = float("nan"), float("inf")                         # rows of no sequence
    out = torch.full((T + extra, hq, 128), 9.0, dtype=dtype, device=DEV)
    got = kb.prompt_attention(q, k, v, SC, cu_seqlens=cu, out=out)
    assert got is out and (out[T:] == 9.0).all()                      # rows behind the last sequence stay
    fresh = kb.prompt_attention(q, k, v, SC, cu_seqlens=cu)
    assert torch.equal(fresh[:T], out[:T]) and (fresh[T:] == 0).all()
    at = 0
    for n in lens:
        if n:
            _check_rows(got[at:at + n], q[at:at + n], k[at:at + n], v[at:at + n], SC, True, (lens, n))
        at += n


def test_packed_pieces(kb):
    """Further pieces: each sequence has more keys than queries (or fewer: its first rows see nothing)."""
    nq, nk = [3, 200, 130, 10], [500, 333, 130, 4]
    q, _, _ = _inputs((sum(nq), 8, 128), (1, 2, 128), torch.bfloat16, 1)
    _, k, v = _inputs((1, 8, 128), (sum(nk), 2, 128), torch.bfloat16, 2)
    cq = torch.tensor([0, 3, 203, 333, 343], dtype=torch.int32, device=DEV)
    ck = torch.tensor([0, 500, 833, 963, 967], dtype=torch.int32, device=DEV)
    got = kb.prompt_attention(q, k, v, SC, cu_seqlens=cq, cu_seqlens_k=ck)
    a = b = 0
    for n, m in zip(nq, nk):
        _check_rows(got[a:a + n], q[a:a + n], k[b:b + m], v[b:b + m], SC, True, (n, m))
        a, b = a + n, b + m
    assert (got[333:339] == 0).all()                                  # 10 queries over 4 keys: six see none


def test_padded_batch(kb):
    q, k, v = _inputs((4, 6, 260, 128), (4, 2, 300, 128), torch.float16, 3)
    ql = torch.tensor([260, 0, 129, 17], dtype=torch.int32, device=DEV)
    kl = torch.tensor([300, 40, 129, 0], dtype=torch.int32, device=DEV)
    for b in range(4):                                                # padding holds garbage
        k[b, :, int(kl[b]):], v[b, :, int(kl[b]):] = float("inf"), float("nan")
    got = kb.prompt_attention(q, k, v, SC, query_lengths=ql, key_lengths=kl)
    for b in range(4):
        n, m = int(ql[b]), int(kl[b])
        assert (got[b, n:] == 0).all()
        if n and m:
            _check_rows(got[b, :n], *(x[b].transpose(0, 1)[:w] for x, w in ((q, n), (k, m), (v, m))), SC, True)
        elif n:
            assert (got[b, :n] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_what_a_row_does_not_see(kb, dtype):
    """Infinities and NaN among later keys and values reach no earlier row, and reach every row that sees them."""
    L = 400
    q, k, v = _inputs((1, 2, L, 128), (1, 1, L, 128), dtype, 4)
    clean = kb.prompt_attention(q, k, v, SC)
    k2, v2 = k.clone(), v.clone()
    v2[0, 0, 150, 5] = float("nan")
    v2[0, 0, 350, 7] = float("inf")
    k2[0, 0, 390] = float("nan")
    got = kb.prompt_attention(q, k2, v2, SC)
    for x in range(2):
        want, mag = attend(q[0, x].double(), k[0, 0].double(), v[0, 0].double(), SC, _limits(L, L, True))
        bound = attention_bound(want, mag, dtype, HALF[dtype], logit_error(q[0, x].double(), k[0, 0].double(), SC))
        off = (got[0, :, x].double() - want).abs()
        assert (off[:150] <= bound[:150]).all()
        others = [c for c in range(128) if c != 5]
        assert (off[150:350][:, others] <= bound[150:350][:, others]).all()
    assert torch.isnan(got[0, 150:390, :, 5]).all()
    assert torch.isinf(got[0, 350:390, :, 7]).all()
    assert torch.isnan(got[0, 390:]).all()
    assert torch.isfinite(clean).all()
    k3 = k.clone()
    k3[0, 0, 3, 9] = float("nan")                                      # every row but the first three
    got = kb.prompt_attention(q, k3, v, SC)
    assert torch.isnan(got[0, 3:]).all() and torch.equal(got[0, :3], clean[0, :3])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,hq,h,Lq,Lk,causal", [(1, 8, 2, 1, 5000, True), (2, 4, 2, 130, 3001, True), (1, 7, 1, 3, 12000, True),
                                                 (1, 4, 4, 257, 2500, False), (1, 1, 1, 700, 600, True)])
def test_few_rows_over_many_keys(kb, dtype, B, hq, h, Lq, Lk, causal):
    """Keys cut in parts and joined: ragged batches, rows that see nothing, values that a row does not see."""
    from kitty_b200 import _lib

    assert _lib.lib().kitty_prompt_workspace_bytes(B, Lq, Lk, hq, h, int(causal), 0) > 0 or Lk < 1000
    q, k, v = _inputs((B, hq, Lq, 128), (B, h, Lk, 128), dtype, Lk)
    got = kb.prompt_attention(q, k, v, SC, causal=causal)
    for b in range(B):
        _check_rows(got[b], *(x[b].transpose(0, 1) for x in (q, k, v)), SC, causal)
    assert torch.equal(kb.prompt_attention(q, k, v, SC, causal=causal), got)
    kl = torch.full((B,), Lk - 70, dtype=torch.int32, device=DEV)
    kl[0] = 5 if B > 1 else Lk - 70
    want = kb.prompt_attention(q[-1:], k[-1:, :, :Lk - 70].contiguous(), v[-1:, :, :Lk - 70].contiguous(), SC, causal=causal)
    k[:, :, Lk - 70:], v[:, :, Lk - 70:] = float("nan"), float("inf")
    got = kb.prompt_attention(q, k, v, SC, causal=causal, key_lengths=kl)
    if B > 1:
        n = Lq - 5                                                     # the first row's queries over five keys
        assert (got[0, :n] == 0).all()
        _check_rows(got[0, n:], q[0, :, n:].transpose(0, 1), k[0, :, :5].transpose(0, 1), v[0, :, :5].transpose(0, 1), SC, True)
    _check_rows(got[-1], q[-1].transpose(0, 1), k[-1, :, :Lk - 70].transpose(0, 1), v[-1, :, :Lk - 70].transpose(0, 1), SC, causal)
    # the same keys in other parts: two roundings of the same numbers
    assert ((got[-1].float() - want[0].float()).abs() <= 4 * HALF[dtype] * v[-1, :, :Lk - 70].float().abs().max()).all()


def test_packed_few_rows_over_many_keys(kb):
    nq, nk = [2, 0, 40], [4000, 100, 6000]
    q, _, _ = _inputs((45, 4, 128), (1, 1, 128), torch.float16, 1)
    _, k, v = _inputs((1, 4, 128), (sum(nk), 1, 128), torch.float16, 2)
    cq = torch.tensor([0, 2, 2, 42], dtype=torch.int32, device=DEV)
    ck = torch.tensor([0, 4000, 4100, 10100], dtype=torch.int32, device=DEV)
    k[4000:4100], v[4000:4100] = float("nan"), float("nan")
    out = torch.full((45, 4, 128), 3.0, dtype=torch.float16, device=DEV)
    kb.prompt_attention(q, k, v, SC, cu_seqlens=cq, cu_seqlens_k=ck, out=out)
    assert (out[42:] == 3.0).all()
    got = kb.prompt_attention(q, k, v, SC, cu_seqlens=cq, cu_seqlens_k=ck)
    assert torch.equal(got[:42], out[:42]) and (got[42:] == 0).all()
    _check_rows(got[:2], q[:2], k[:4000], v[:4000], SC, True)
    _check_rows(got[2:42], q[2:42], k[4100:], v[4100:], SC, True)


def test_extreme_logits(kb):
    """Maxima that rise and fall by far more than the lag, and rows whose weight sits on one key."""
    L = 520
    q, k, v = _inputs((1, 2, L, 128), (1, 1, L, 128), torch.bfloat16, 5, qscale=6.0)
    ramp = torch.linspace(0.05, 4.0, L, device=DEV)[None, None, :, None]
    for kk in ((k.float() * ramp).bfloat16(), (k.float() * ramp.flip(2)).bfloat16()):
        got = kb.prompt_attention(q, kk, v, SC)
        _check_rows(got[0], q[0].transpose(0, 1), kk[0].transpose(0, 1), v[0].transpose(0, 1), SC, True)
    zero = torch.zeros_like(q)
    got = kb.prompt_attention(zero, k, v, SC)                          # all weights equal: running means
    _check_rows(got[0], zero[0].transpose(0, 1), k[0].transpose(0, 1), v[0].transpose(0, 1), SC, True)


def test_streams_graphs_and_empty(kb):
    q, k, v = _inputs((1, 4, 200, 128), (1, 2, 200, 128), torch.float16, 6)
    want = kb.prompt_attention(q, k, v, SC)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:                                                  # two calls at once
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append([kb.prompt_attention(q, k, v, SC) for _ in range(3)])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for per in outs for o in per)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = kb.prompt_attention(q, k, v, SC)
    q.copy_(q.flip(2))
    graph.replay()
    assert torch.equal(cap, kb.prompt_attention(q, k, v, SC))
    assert kb.prompt_attention(q[:, :, :0], k, v, SC).shape == (1, 0, 4, 128)
    assert kb.prompt_attention(q[:0], k[:0], v[:0], SC).shape == (0, 200, 4, 128)
    none = kb.prompt_attention(q, k[:, :, :0], v[:, :, :0], SC, causal=False)
    assert (none == 0).all()
    one = kb.prompt_attention(q, k[:, :1].expand(1, 4, 200, 128), v[:, :1].expand(1, 4, 200, 128), SC)
    assert torch.equal(one, kb.prompt_attention(q, k[:, :1], v[:, :1], SC))


def test_agrees_with_decode_attention(kb):
    """The row of a prompt's last token equals decode attention over a cache that still holds everything in fp16."""
    import types

    cfg = types.SimpleNamespace(num_hidden_layers=1, head_dim=128, num_key_value_heads=2, num_attention_heads=8, hidden_size=1024)
    q, k, v = _inputs((2, 8, 150, 128), (2, 2, 150, 128), torch.float16, 8)
    cache = kb.KittyCache(cfg, 2, 256, device=DEV)
    cache.update(k, v, 0)
    cache.quantize_prefill(0)
    assert cache.kv_cache[0].PageCount_K == 0                           # 150 tokens: sink and Q-buffer only
    dec = kb.decode_attention(q[:, :, -1:].contiguous(), cache.kv_cache[0], 2, SC)
    got = kb.prompt_attention(q, k, v, SC)[:, -1:]
    for b in range(2):
        for x in range(8):
            qx, kx, vx = q[b, x, -1:].double(), k[b, x // 4].double(), v[b, x // 4].double()
            want, mag = attend_fast(qx, kx, vx, SC, torch.tensor([150], device=DEV))
            bound = attention_bound(want, mag, torch.float16, HALF[torch.float16], logit_error(qx, kx, SC))
            assert ((got[b, :, x].double() - want).abs() <= bound).all()
    assert (dec.float() - got.float()).abs().max() <= 1e-2 * got.float().abs().max()


def test_rows_off_their_boundaries_and_other_orders(kb):
    """Views whose rows start anywhere, channels apart, heads expanded: read through a copy, the same result."""
    q, k, v = _inputs((1, 4, 90, 128), (1, 2, 90, 128), torch.bfloat16, 9)
    want = kb.prompt_attention(q, k, v, SC)

    def off(x, pad):
        wide = torch.zeros(*x.shape[:-1], 128 + pad, dtype=x.dtype, device=DEV)
        wide[..., pad:] = x
        return wide[..., pad:]

    assert torch.equal(kb.prompt_attention(off(q, 1), off(k, 3), off(v, 4), SC), want)
    apart = torch.stack((q, q), -1)[..., 0]
    assert apart.stride(-1) == 2 and torch.equal(kb.prompt_attention(apart, k, v, SC), want)
    cu = torch.tensor([0, 90], dtype=torch.int32, device=DEV)
    packed = [off(x[0].transpose(0, 1).contiguous(), 2) for x in (q, k, v)]
    assert torch.equal(kb.prompt_attention(*packed, SC, cu_seqlens=cu), want[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_patched_model_takes_the_prompt_kernel(kb, dtype, monkeypatch):
    """patch_model(prompt_kernel=True): every layer's prompt goes through the operator, whose results meet the formula;
    float32 models and masked batches keep torch's attention."""
    from transformers import LlamaConfig, LlamaForCausalLM

    from kitty_b200 import hf_adapter

    torch.manual_seed(0)
    cfg = LlamaConfig(hidden_size=512, intermediate_size=1024, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                      head_dim=128, vocab_size=1000, max_position_embeddings=4096)
    model = LlamaForCausalLM(cfg).eval().to(dtype).to(DEV)
    assert hf_adapter.patch_model(model, prompt_kernel=True) == 2
    calls = []

    def recorded(q, k, v, scaling):
        out = kb.prompt_attention(q, k, v, scaling)
        calls.append((q, k, v, scaling, out))
        return out

    monkeypatch.setattr(hf_adapter, "prompt_attention", recorded)
    ids = torch.randint(0, 1000, (2, 150), device=DEV)
    cache = kb.get_kvcache_kitty(cfg, 2, 512, device=DEV)
    toks = hf_adapter.greedy_decode(model, ids, 4, cache)
    assert toks.shape == (2, 4) and len(calls) == 2 and cache.get_seq_length() == 153
    for q, k, v, scaling, out in calls:
        for b in range(2):
            _check_rows(out[b], *(x[b].transpose(0, 1) for x in (q, k, v)), scaling, True)
    single = LlamaForCausalLM(cfg).eval().to(DEV)
    hf_adapter.patch_model(single, prompt_kernel=True)
    hf_adapter.greedy_decode(single, ids, 2, kb.get_kvcache_kitty(cfg, 2, 512, device=DEV))
    assert len(calls) == 2


def _best_us(call, n=5):
    """Shortest of n timed calls (after one that is not)."""
    call()
    best = float("inf")
    for _ in range(n):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        call()
        b.record()
        b.synchronize()
        best = min(best, 1000.0 * a.elapsed_time(b))
    return best


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
def test_padding_that_is_not_finite_costs_no_more(kb, dtype, causal):
    """Keys and values behind a row's last one, or of the next sequence: the same bits in about the same time, whatever they
    hold.  (The limit is wide: a row computed without the tensor cores takes thousands of times as long.)"""
    q, k, v = _inputs((2, 8, 2500, 128), (2, 2, 2500, 128), dtype, 21)
    lens = torch.tensor([2450, 1111], dtype=torch.int32, device=DEV)
    k2, v2 = k.clone(), v.clone()
    for b in range(2):
        n = int(lens[b])
        k[b, :, n:], v[b, :, n:] = 0.0, 0.0
        k2[b, :, n:], v2[b, :, n:] = float("inf"), float("nan")
    run = lambda kk, vv: kb.prompt_attention(q, kk, vv, SC, causal=causal, key_lengths=lens)  # noqa: E731
    assert torch.equal(run(k2, v2), run(k, v))
    assert _best_us(lambda: run(k2, v2)) <= 3.0 * _best_us(lambda: run(k, v)) + 200.0
    # packed: the second sequence is not finite, the first does not notice
    qp, kp, vp = (x[0].transpose(0, 1).contiguous() for x in (q, k, v))
    cu = torch.tensor([0, 1300, 2500], dtype=torch.int32, device=DEV)
    packed = lambda vv: kb.prompt_attention(qp, kp, vv, SC, causal=causal, cu_seqlens=cu)  # noqa: E731
    bad = vp.clone()
    bad[1300:] = float("-inf")
    want, got = packed(vp), packed(bad)
    assert torch.equal(got[:1300], want[:1300]) and not torch.isfinite(got[1300:]).any()
    assert _best_us(lambda: packed(bad)) <= 3.0 * _best_us(lambda: packed(vp)) + 2000.0
    assert kb.prompt_attention_status(DEV) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,h,Lq,Lk", [(1, 1, 700, 700), (6, 2, 300, 333), (3, 1, 40, 3000), (2, 2, 260, 200)])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(kb, dtype, hq, h, Lq, Lk):
    """Infinities and NaN at the edges of tiles and within them: a row that sees some gets their sum in their channels, and
    otherwise every row has the bits that it has with zeros in their place."""
    inf, nan = float("inf"), float("nan")
    q, k, v = _inputs((1, hq, Lq, 128), (1, h, Lk, 128), dtype, 22)
    odd = torch.zeros(h, Lk, 128, device=DEV, dtype=torch.float64)
    for x in range(h):
        for i, key in enumerate([0, 63, 127, 128, 129, 255, 256, 300, Lk - 130, Lk - 3, Lk - 2, Lk - 1]):
            if 0 <= key < Lk:
                odd[x, key, (7 * i + x) % 128] = (nan, inf, -inf)[i % 3]
        odd[x, Lk // 2, 3], odd[x, Lk - 5, 3] = inf, -inf                  # opposite ones: NaN from the second on
        odd[x, Lk - 9] = nan                                             # a whole row
    hit = odd != 0
    v = torch.where(hit[None], torch.zeros_like(v), v)
    want = kb.prompt_attention(q, k, v, SC)
    got = kb.prompt_attention(q, k, torch.where(hit[None], odd[None].to(dtype), v), SC)
    lim = _limits(Lq, Lk, True)
    reach = torch.cat((torch.zeros(h, 1, 128, device=DEV, dtype=torch.float64), odd.cumsum(1)), 1)[:, lim]    # [h, Lq, 128]
    for x in range(hq):
        add = reach[x // (hq // h)]
        w, g = want[0, :, x], got[0, :, x]
        assert torch.equal(g[add == 0], w[add == 0])
        assert torch.isnan(g[torch.isnan(add)]).all()
        assert (g[torch.isinf(add)].double() == add[torch.isinf(add)]).all()
    assert torch.isfinite(want).all() and kb.prompt_attention_status(DEV) == 0


def test_nothing_but_nan(kb):
    """Values that are all NaN: every row that sees one is NaN, in a bounded time."""
    q, k, v = _inputs((1, 8, 3000, 128), (1, 2, 3000, 128), torch.bfloat16, 23)
    clean = _best_us(lambda: kb.prompt_attention(q, k, v, SC), 2)
    v[:] = float("nan")
    assert torch.isnan(kb.prompt_attention(q, k, v, SC)).all()
    assert _best_us(lambda: kb.prompt_attention(q, k, v, SC), 2) <= 20.0 * clean + 5000.0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_blocks_that_take_several_items_of_several_tiles(kb, dtype):
    """More items than multiprocessors, each of several key tiles, of unequal numbers: what a block carries from item to item."""
    q, k, v = _inputs((3, 24, 1400, 128), (3, 12, 1400, 128), dtype, 24)
    ql = torch.tensor([1400, 900, 1400], dtype=torch.int32, device=DEV)
    kl = torch.tensor([1400, 900, 130], dtype=torch.int32, device=DEV)
    got = kb.prompt_attention(q, k, v, SC, query_lengths=ql, key_lengths=kl)
    for b in range(3):
        n, m = int(ql[b]), int(kl[b])
        assert (got[b, n:] == 0).all()
        _check_rows(got[b, :n], q[b, :, :n].transpose(0, 1), k[b, :, :m].transpose(0, 1), v[b, :, :m].transpose(0, 1), SC, True)
    again = kb.prompt_attention(q, k, v, SC, query_lengths=ql, key_lengths=kl)
    assert torch.equal(got, again)                                     # and the same bits each time
    lens = [1400, 3, 700, 129, 1, 1399]
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
    qp, kp, vp = _inputs((sum(lens), 24, 128), (sum(lens), 12, 128), dtype, 25)
    got = kb.prompt_attention(qp, kp, vp, SC, cu_seqlens=cu, causal=False)
    for a, b in zip(cu[:-1].tolist(), cu[1:].tolist()):
        _check_rows(got[a:b], qp[a:b], kp[a:b], vp[a:b], SC, False, (a, b))
    assert kb.prompt_attention_status(DEV) == 0


def test_outputs_over_the_inputs_are_refused(kb):
    """Other rows still read what an output would overwrite; slices of one buffer that only lie between each other are fine."""
    q, k, v = _inputs((2, 4, 300, 128), (2, 4, 300, 128), torch.float16, 26)
    want = kb.prompt_attention(q, k, v, SC)
    wide = torch.zeros(2, 300, 12, 128, dtype=torch.float16, device=DEV)
    for i, x in enumerate((q, k, v)):
        wide[:, :, 4 * i:4 * i + 4] = x.transpose(1, 2)
    a, b, c = (wide[:, :, 4 * i:4 * i + 4].transpose(1, 2) for i in range(3))
    assert torch.equal(kb.prompt_attention(a, b, c, SC), want)
    for i in range(3):
        args = [q, k, v]
        out = args[i].clone()                                           # [B, H, T, 128] in memory, taken as [B, T, H, 128]
        args[i] = out
        with pytest.raises(ValueError, match="overlaps"):
            kb.prompt_attention(*args, SC, out=out.view(2, 300, 4, 128))
        assert torch.equal(args[i], (q, k, v)[i])
    cu = torch.tensor([0, 300], dtype=torch.int32, device=DEV)
    kp, vp = k[0].transpose(0, 1), v[0].transpose(0, 1)
    pool = torch.empty(600, 4, 128, dtype=torch.float16, device=DEV)
    pool[:300] = q[0].transpose(0, 1)
    with pytest.raises(ValueError, match="overlaps"):
        kb.prompt_attention(pool[:300], kp, vp, SC, cu_seqlens=cu, out=pool[299:599])
    got = kb.prompt_attention(pool[:300], kp, vp, SC, cu_seqlens=cu, out=pool[300:])
    assert torch.equal(got, want[0])


def test_patched_model_reports_a_wait_that_ran_out(kb):
    """Once per prompt the patched model looks at the status word that the kernels set when they give up."""
    from transformers import LlamaConfig, LlamaForCausalLM

    from kitty_b200 import hf_adapter, prompt

    cfg = LlamaConfig(hidden_size=256, intermediate_size=256, num_hidden_layers=3, num_attention_heads=2, num_key_value_heads=1,
                      head_dim=128, vocab_size=100, max_position_embeddings=512)
    model = LlamaForCausalLM(cfg).eval().bfloat16().to(DEV)
    hf_adapter.patch_model(model, prompt_kernel=True)
    assert [m.self_attn.kitty_prompt_check for m in model.model.layers] == [False, False, True]
    ids = torch.randint(0, 100, (1, 70), device=DEV)
    run = lambda: hf_adapter.greedy_decode(model, ids, 2, kb.get_kvcache_kitty(cfg, 1, 256, device=DEV))  # noqa: E731
    run()
    word = prompt._status[torch.device(DEV)]
    word.fill_(1)
    try:
        with pytest.raises(kb.KittyError, match="prompt_attention on cuda:0"):
            run()
    finally:
        word.zero_()
    run()
    hf_adapter.patch_model(model)                                     # torch's attention: nothing to look at
    word.fill_(1)
    try:
        run()
    finally:
        word.zero_()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("margin", [4.0, 12.0, 18.0, 20.0])
def test_many_small_weights_behind_a_large_one(kb, dtype, margin):
    """One key far above 32767 equal ones, whose values alone are not zero: the result is all theirs,
    n w / (1 + n w) with w = e^-margin."""
    from kitty_b200 import _lib

    hq, Lq, n = 16, 4096, 32767
    assert _lib.lib().kitty_prompt_workspace_bytes(1, Lq, n + 1, hq, 1, 0, 0) == 0      # keys not cut in parts
    q = torch.zeros(1, hq, Lq, 128, dtype=dtype, device=DEV)
    q[..., 7] = 1.0
    k, v = torch.zeros(1, 1, n + 1, 128, dtype=dtype, device=DEV), torch.ones(1, 1, n + 1, 128, dtype=dtype, device=DEV)
    k[:, :, 0, 7], v[:, :, 0] = margin, 0.0
    got = kb.prompt_attention(q, k, v, 1.0, causal=False)
    w = torch.tensor(-margin, dtype=torch.float64).exp().item()
    want = n * w / (1.0 + n * w)
    # a weight is rounded to half a step, or to half of 2^-31 of the largest where that is more (fp16's smallest number is
    # 2^-24, and the largest weight 2^7); logits and exponentials are off by 2^-16 of the weight at most; the output's half step
    part = max(HALF[dtype], 2.0 ** -32 / w if dtype == torch.float16 else 0.0) + 2.0 ** -16
    assert (got.double() - want).abs().max().item() <= want * (part + HALF[dtype] * (1.0 + part))


@pytest.mark.parametrize("hq", [1, 2])
def test_an_item_that_takes_longer_than_a_wait_may(kb, hq):
    """One row over 2^28 keys (rows of a small buffer, 16 bytes apart) that are not cut in parts: some two million key tiles in
    a row, over two seconds, during which those who wait for the item's end wait on."""
    from kitty_b200 import _lib

    n = (1 << 28) - 5
    buf = torch.zeros(8 * n + 120, dtype=torch.bfloat16, device=DEV)
    buf[-928:] = 1.0                                                    # the last 101 rows are all ones, their logits 45
    k = buf.as_strided((1, 1, n, 128), (8 * n, 8 * n, 8, 1))
    q = torch.full((1, hq, 1, 128), 4.0, dtype=torch.bfloat16, device=DEV)
    out = torch.zeros(1, 1, hq, 128, dtype=torch.bfloat16, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    st = [_lib.head_rows(x, repeated=False) for x in (q, k, k)]
    assert all(a is b for (a, _), b in zip(st, (q, k, k)))
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    _lib.call_on(q.device, _lib.lib().kitty_prompt_attn, "kitty_prompt_attn", q.data_ptr(), k.data_ptr(), k.data_ptr(), _lib.KITTY_BF16,
                 _lib.i64_array(st[0][1] + st[1][1] + st[2][1]), 1, 1, n, hq, 1, SC, 1, None, None, None, None, out.data_ptr(), 1,
                 status.data_ptr(), None, 0)
    b.record()
    b.synchronize()
    # the rows before those, whose first channels are zero, have a 17th of the weight and less: 1 - 0.0006 and up
    assert int(status.item()) == 0 and (out == 1.0).all()
    assert a.elapsed_time(b) > 2000.0, a.elapsed_time(b)                # the case in the name
