"""The 8-bit cache: what is stored, and attention over it, against plain 64-bit forms."""
import pytest
import torch

from tests.ops_ref import HALF, attend_fast, attention_bound, held_values, hold, logit_error, read_records, rotate

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SC = 128 ** -0.5


@pytest.fixture(scope="module")
def kb():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import kitty_b200

    return kitty_b200


def _kv(B, H, T, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    k = torch.randn(B, T, H, 128, generator=g, device=DEV)
    k[..., :4] *= 8.0
    v = torch.randn(B, T, H, 128, generator=g, device=DEV)
    return k.to(dtype).transpose(1, 2), v.to(dtype).transpose(1, 2)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _scattered(B, pages, seed=0):
    return torch.randperm(B * pages, generator=torch.Generator().manual_seed(seed)).view(B, pages).to(DEV)


def _held(x, n, dtype):
    """Tokens [H, n, 128] as the cache gives them back: whole blocks rounded to codes, the open block as it was."""
    full = n // 32 * 32
    return torch.cat((held_values(x[:, :full], dtype), x[:, full:n]), 1)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H", [1, 3])
@pytest.mark.parametrize("T", [1, 31, 32, 33, 160, 261])
def test_append_and_expand(kb, dtype, H, T):
    B = 2
    k, v = _kv(B, H, T, dtype, T)
    layer = kb.KV8Layer(B, 300, H, dtype=dtype, device=DEV, page_table=_scattered(B, 3))
    zero, n = _i32([0, 0]), _i32([T, T // 2])
    kb.kv8_append(layer, k, v, zero, lengths=n)
    ke, ve = kb.kv8_expand(layer, n, T + 5)
    for b, m in enumerate([T, T // 2]):
        assert torch.equal(ke[b, :, :m], _held(k[b], m, dtype)) and torch.equal(ve[b, :, :m], _held(v[b], m, dtype))
        assert (ke[b, :, m:] == 0).all() and (ve[b, :, m:] == 0).all()
    for b, (kc, ks, vc, vs) in enumerate(read_records(layer, [T, T // 2])):
        full = kc.shape[1]
        for got, gs, x in ((kc, ks, k[b]), (vc, vs, v[b])):
            codes, scale = hold(x[:, :full].cpu())
            assert torch.equal(got, codes.reshape(H, full, 128)) and torch.equal(gs, scale.float())
    layer.check()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout,r", [("half", 128), ("half", 64), ("half", 20), ("interleaved", 128), ("interleaved", 64),
                                      ("interleaved", 20)])
def test_same_bytes_however_the_tokens_are_cut(kb, dtype, layout, r):
    B, H, hq, T = 2, 2, 6, 150
    k, v = _kv(B, H, T, dtype, r)
    q = torch.randn(B, hq, T, 128, device=DEV).to(dtype)
    rot = kb.RotaryEmbedding(rotary_dim=r, layout=layout, device=DEV)
    first = _i32([7, 64])                                      # what the rows hold before
    k0, v0 = _kv(B, H, 64, dtype, 99)
    table = _scattered(B, 2, 5)
    layers = [kb.KV8Layer(B, 256, H, dtype=dtype, device=DEV, page_table=table) for _ in range(4)]
    for lay in layers:
        kb.kv8_append(lay, k0, v0, torch.zeros_like(first), lengths=first, rotary=rot)
    whole = kb.kv8_append(layers[0], k, v, first, rotary=rot, query=q)
    parts = []
    for a, b in ((0, 1), (1, 26), (26, 26), (26, 90), (90, 91), (91, 150)):
        parts.append(kb.kv8_append(layers[1], k[:, :, a:b], v[:, :, a:b], first + a, rotary=rot, query=q[:, :, a:b]))
    for t in range(T):
        kb.kv8_append(layers[2], k[:, :, t:t + 1], v[:, :, t:t + 1], first + t, rotary=rot)
    # turned by its own call first, then appended as it is
    pos = first.long()[:, None] + torch.arange(T, device=DEV)
    rq, rk = kb.apply_rotary(q, k, pos, rot)
    kb.kv8_append(layers[3], rk, v, first)
    assert torch.equal(torch.cat(parts, 2), whole) and torch.equal(whole, rq)
    for lay in layers[1:]:
        for name in ("pages", "tail_k", "tail_v"):
            x, y = getattr(lay, name), getattr(layers[0], name)
            if name == "pages":
                assert torch.equal(x, y)
            else:
                for b in range(B):                              # the open block's tokens; older ones may differ
                    m = (int(first[b]) + T) % 32
                    assert torch.equal(x[b, :, :m], y[b, :, :m])
        lay.check()


def test_rotated_keys_against_the_formula(kb):
    """A rotated key is its 64-bit value to half a step before it is stored: the open block shows it."""
    dtype = torch.bfloat16
    k, v = _kv(1, 2, 30, dtype, 3)
    rot = kb.RotaryEmbedding(base=500000.0, rotary_dim=96, device=DEV)
    layer = kb.KV8Layer(1, 4096, 2, dtype=dtype, device=DEV)
    kb.kv8_append(layer, k, v, _i32([4032]), rotary=rot)
    want = rotate(k, 4032 + torch.arange(30, device=DEV)[None], rot.inv_freq.to(DEV), 1.0, 96, "half")
    got, vals = kb.kv8_expand(layer, _i32([4062]), 30, start=_i32([4032]))
    assert ((got.double() - want).abs() <= HALF[dtype] * want.abs() + 2.0 ** -20 * 40.0).all() and torch.equal(vals, v)


def test_special_values(kb):
    """Zeros, one number, halves between codes, subnormals, the type's largest; an infinity or NaN marks its block."""
    for dtype in (torch.float16, torch.bfloat16):
        tops = [127.0, 254.0, 1.0, float(torch.finfo(dtype).max), float(torch.finfo(dtype).tiny),
                float(torch.finfo(dtype).smallest_normal) * float(torch.finfo(dtype).eps), 0.0]
        k = torch.zeros(1, 1, 32 * len(tops), 128, dtype=dtype, device=DEV)
        for i, top in enumerate(tops):
            blk = torch.linspace(-1, 1, 32 * 128, device=DEV, dtype=torch.float64) * top
            if top in (127.0, 254.0):
                blk = torch.round(blk * 2) / 2                  # many exact halves
            k[0, 0, 32 * i:32 * i + 32] = blk.to(dtype).view(32, 128)
            if top:
                k[0, 0, 32 * i, 0] = top
        layer = kb.KV8Layer(1, 256, 1, dtype=dtype, device=DEV)
        n = _i32([k.shape[2]])
        kb.kv8_append(layer, k, -k, _i32([0]))
        ke, ve = kb.kv8_expand(layer, n, k.shape[2])
        assert torch.equal(ke[0], _held(k[0], k.shape[2], dtype)) and torch.equal(ve[0], _held(-k[0], k.shape[2], dtype))
        bad = k.clone()
        bad[0, 0, 40, 3], bad[0, 0, 70, 9] = float("inf"), float("nan")
        kb.kv8_append(layer, bad, k, _i32([0]))
        ke, _ = kb.kv8_expand(layer, n, k.shape[2])
        assert torch.isnan(ke[0, 0, 32:96]).all()
        assert torch.equal(ke[0, 0, 96:], _held(k[0], k.shape[2], dtype)[0, 96:])


def _attention_check(got, q, layer, lengths, tails, scaling):
    """Against the record's own codes and scales in 64 bits (the open block's 16-bit tokens as given)."""
    B, hq = q.shape[:2]
    G = hq // layer.H_KV
    for b, (kc, ks, vc, vs) in enumerate(read_records(layer, lengths)):
        n = lengths[b]
        if n == 0:
            assert (got[b] == 0).all()
            continue
        full = n // 32 * 32
        kk = (kc.view(layer.H_KV, -1, 32, 128) * ks.double()[..., None, None]).reshape(layer.H_KV, full, 128)
        vv = (vc.view(layer.H_KV, -1, 32, 128) * vs.double()[..., None, None]).reshape(layer.H_KV, full, 128)
        kk = torch.cat((kk.to(DEV), tails[0][b][:, full:n].double()), 1)
        vv = torch.cat((vv.to(DEV), tails[1][b][:, full:n].double()), 1)
        for x in range(hq):
            qx, kx, vx = q[b, x].double(), kk[x // G], vv[x // G]
            want, mag = attend_fast(qx, kx, vx, scaling, torch.tensor([n], device=DEV))
            # query elements are within half of (largest of the head) / 32512 of their value, 2^-15.98 of the largest
            delta = logit_error(qx, kx, scaling) + 2.0 ** -15.9 * (qx.abs().max() * kx.abs().sum(1).max()).item() * abs(scaling)
            # weights within the same part of their block's largest; those of the open block are sums of two 16-bit numbers
            # (2^-16 of their own size)
            bound = attention_bound(want, mag, q.dtype, 2.0 ** -16, delta)
            if full:
                p = torch.softmax((kx @ qx[0]) * scaling, 0)[:full].view(-1, 32)
                share = p.amax(1) @ vx[:full].abs().view(-1, 32, 128).sum(1)
                bound = bound + 2.0 ** -15.9 * share * (1.0 + 2.0 * delta)
            off = (got[b, :, x].double() - want).abs()
            assert (off <= bound).all(), (b, x, n, off.max().item(), bound.max().item())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,hq", [(1, 1), (2, 8), (1, 7), (1, 8), (2, 18), (1, 16)])
@pytest.mark.parametrize("room", [0, 4100])
@pytest.mark.parametrize("lengths", [[1], [31, 32, 33], [0, 517, 64, 0, 130], [1700], [1024, 992]])
def test_attention(kb, dtype, H, hq, lengths, room):
    """room: caches with place for short rows only and for long ones go different ways."""
    B, L = len(lengths), max(lengths) + room
    k, v = _kv(B, H, max(lengths), dtype, max(lengths) + hq)
    q = (0.7 * torch.randn(B, hq, 1, 128, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)).to(dtype)
    layer = kb.KV8Layer(B, L, H, dtype=dtype, device=DEV, page_table=_scattered(B, -(-L // 128)))
    n = _i32(lengths)
    layer.tail_k.fill_(float("nan"))                           # stale tokens of open blocks hold anything
    layer.tail_v.fill_(float("inf"))
    kb.kv8_append(layer, k, v, torch.zeros_like(n), lengths=n)
    got = kb.kv8_attention(q, layer, n, SC)
    assert got.shape == (B, 1, hq, 128)
    _attention_check(got, q, layer, lengths, (k, v), SC)
    out = torch.empty_like(got)
    assert kb.kv8_attention(q, layer, n, SC, out=out) is out and torch.equal(out, got)       # the same bits again
    layer.check()


@pytest.mark.parametrize("cap", [256, 1280, 4224])
def test_attention_many_short_rows(kb, cap):
    """More rows than multiprocessors, in caches with place for a little and for more."""
    dtype, B = torch.float16, 90
    lengths = [(53 * i) % 257 for i in range(B)]
    layer = kb.KV8Layer(B, cap, 2, dtype=dtype, device=DEV, page_table=_scattered(B, cap // 128))
    k, v = _kv(B, 2, 256, dtype, 3)
    n = _i32(lengths)
    kb.kv8_append(layer, k, v, torch.zeros_like(n), lengths=n)
    q = torch.randn(B, 14, 1, 128, device=DEV).to(dtype)
    _attention_check(kb.kv8_attention(q, layer, n, SC), q, layer, lengths, (k, v), SC)
    layer.check()


def test_attention_many_rows_and_a_long_one(kb):
    dtype = torch.bfloat16
    lengths = [3, 0, 9000] + [(37 * i) % 200 for i in range(147)]
    B = len(lengths)
    layer = kb.KV8Layer(B, 9000, 2, dtype=dtype, device=DEV, num_pages=400,
                        page_table=torch.zeros(B, 71, dtype=torch.int64, device=DEV))
    at = 0
    for b, n in enumerate(lengths):                             # rows share a pool of pages
        m = -(-n // 128)
        layer.page_table[b, :m] = torch.arange(at, at + m, device=DEV)
        at += m
    assert at <= 400
    k, v = _kv(B, 2, 200, dtype, 1)
    n = _i32(lengths)
    short = n.clamp(max=200)
    kb.kv8_append(layer, k, v, torch.zeros_like(n), lengths=short)
    kl, vl = _kv(1, 2, 8800, dtype, 2)
    more = torch.zeros_like(n)
    more[2] = 8800
    kb.kv8_append(layer, kl.expand(B, -1, -1, -1), vl.expand(B, -1, -1, -1), short, lengths=more)
    q = torch.randn(B, 8, 1, 128, device=DEV).to(dtype)
    got = kb.kv8_attention(q, layer, n, SC)
    ks = [k[b] for b in range(B)]
    vs = [v[b] for b in range(B)]
    ks[2], vs[2] = torch.cat((k[2], kl[0]), 1), torch.cat((v[2], vl[0]), 1)
    _attention_check(got, q, layer, lengths, (ks, vs), SC)


def test_query_scales(kb):
    """Queries far outside fp16's range, tiny ones and zeros."""
    k, v = _kv(4, 1, 70, torch.bfloat16, 6)
    layer = kb.KV8Layer(4, 128, 1, dtype=torch.bfloat16, device=DEV)
    kb.kv8_append(layer, k, v, _i32([0] * 4))
    q = torch.randn(4, 4, 1, 128, device=DEV)
    q *= torch.tensor([1e20, 1e-20, 0.0, 1.0], device=DEV)[:, None, None, None]
    q = q.bfloat16()
    for b, sc in enumerate((SC * 1e-20, SC * 1e20, SC, SC)):
        got = kb.kv8_attention(q[b:b + 1], _row_view(layer, b), _i32([70]), sc)
        _attention_check(got, q[b:b + 1], _row_view(layer, b), [70], (k[b:b + 1], v[b:b + 1]), sc)


def _row_view(layer, b):
    """A cache of one row over the same pages."""
    import copy

    one = copy.copy(layer)
    one.MAX_BS = 1
    one.page_table = layer.page_table[b:b + 1].contiguous()
    one.tail_k, one.tail_v = layer.tail_k[b:b + 1], layer.tail_v[b:b + 1]
    one._workspace_need, one._c_layer = {}, None
    return one


def test_bad_pages_and_lengths_are_skipped_and_reported(kb):
    layer = kb.KV8Layer(2, 256, 1, device=DEV, num_pages=4)
    k, v = _kv(2, 1, 256, torch.bfloat16, 9)
    kb.kv8_append(layer, k, v, _i32([0, 0]))
    before = layer.pages.clone()
    layer.check()
    layer.page_table[1, 1] = 4
    kb.kv8_append(layer, k.flip(2), v, _i32([128, 128]), lengths=_i32([0, 128]))
    assert torch.equal(layer.pages, before)
    with pytest.raises(ValueError, match="page-table"):
        layer.check()
    q = torch.randn(2, 4, 1, 128, device=DEV).bfloat16()
    got = kb.kv8_attention(q, layer, _i32([256, 256]), SC)
    half = kb.kv8_attention(q, layer, _i32([256, 128]), SC)
    assert torch.equal(got[0], half[0]) and torch.isfinite(got).all()
    ke, _ = kb.kv8_expand(layer, _i32([256, 256]), 256)
    assert (ke[1, :, 128:] == 0).all()
    layer.page_table[1, 1] = -1
    kb.kv8_attention(q, layer, _i32([256, 256]), SC)
    layer.page_table[1, 1] = 3
    layer.status.zero_()
    tails = layer.tail_k.clone()
    for start, n in (([0, 250], [0, 10]), ([-1, 0], [5, 0]), ([300, 0], [1, 0]), ([0, 0], [0, -3]), ([0, 0], [0, 999])):
        layer.status.zero_()
        kb.kv8_append(layer, k[:, :, :10], v[:, :, :10], _i32(start), lengths=_i32(n))
        with pytest.raises(ValueError, match="length"):
            layer.check()
    del tails
    layer.status.zero_()
    assert kb.kv8_attention(q, layer, _i32([500, -2]), SC).shape == (2, 1, 4, 128)
    with pytest.raises(ValueError, match="length"):
        layer.check()


def test_steps_from_a_graph(kb):
    """Append with rotation, attention and the length's own increment captured once and replayed across a block's and a
    page's end; two graphs with their own caches side by side."""
    dtype, B, H, hq, L0 = torch.float16, 2, 2, 8, 120
    rot = kb.RotaryEmbedding(device=DEV)

    def fresh():
        lay = kb.KV8Layer(B, 512, H, dtype=dtype, device=DEV)
        k, v = _kv(B, H, L0, dtype, 1)
        n = _i32([L0, L0 - 50])
        kb.kv8_append(lay, k, v, torch.zeros_like(n), lengths=n, rotary=rot)
        return lay, n

    toks = [(_kv(B, H, 1, dtype, 100 + i), torch.randn(B, hq, 1, 128, device=DEV).to(dtype)) for i in range(45)]

    def step(lay, n, kt, vt, q):
        rq = kb.kv8_append(lay, kt, vt, n, rotary=rot, query=q)
        n += 1
        return kb.kv8_attention(rq, lay, n, SC)

    lay, n = fresh()
    want = [step(lay, n, kt, vt, q) for (kt, vt), q in toks]
    runs = []
    for _ in range(2):
        lay2, n2 = fresh()
        kt, vt, q = toks[0][0][0].clone(), toks[0][0][1].clone(), toks[0][1].clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(lay2, n2, kt, vt, q)
        runs.append((lay2, n2, kt, vt, q, g, out))
    for i, ((k1, v1), q1) in enumerate(toks):
        for lay2, n2, kt, vt, q, g, out in runs:
            kt.copy_(k1), vt.copy_(v1), q.copy_(q1)
            g.replay()
            assert torch.equal(out, want[i]), i
    assert torch.equal(runs[0][0].pages, lay.pages)


def test_prompt_then_tokens_then_a_further_piece(kb):
    """The operators as they are used together: rotate, attend and store a prompt; decode; attend a further piece over
    the expanded cache."""
    dtype, B, H, hq, L = torch.bfloat16, 2, 2, 8, 200
    rot = kb.RotaryEmbedding(base=500000.0, device=DEV)
    layer = kb.KV8Layer(B, 512, H, dtype=dtype, device=DEV, page_table=_scattered(B, 4))
    g = torch.Generator(device=DEV).manual_seed(11)
    mk = lambda h, t: torch.randn(B, t, h, 128, generator=g, device=DEV).to(dtype).transpose(1, 2)  # noqa: E731
    q, k, v = mk(hq, L), mk(H, L), mk(H, L)
    lens = _i32([L, 77])
    pos = torch.arange(L, device=DEV)
    rq, rk = kb.apply_rotary(q, k, pos, rot)
    prompt = kb.prompt_attention(rq, rk, v, SC, query_lengths=lens, key_lengths=lens)
    kb.kv8_append(layer, rk, v, torch.zeros_like(lens), lengths=lens)
    n = lens.clone()
    for i in range(3):                                              # tokens
        qt, kt, vt = mk(hq, 1), mk(H, 1), mk(H, 1)
        rqt = kb.kv8_append(layer, kt, vt, n, rotary=rot, query=qt)
        n += 1
        out = kb.kv8_attention(rqt, layer, n, SC)
    ke, ve = kb.kv8_expand(layer, n, L + 3)
    same = kb.prompt_attention(rqt, ke, ve, SC, key_lengths=n)      # one query over the same tokens
    # the same codes, in the prompt kernel rounded to bf16 first: half a step each of keys, values and weights
    size = (rqt.double().abs() @ ke.double().abs().repeat_interleave(hq // H, 1).transpose(2, 3)).max().item() * SC
    bound = (3 * 2.0 ** -8 + 2 * 2.0 ** -8 * size) * ve.double().abs().max().item()
    assert (same.double() - out.double()).abs().max().item() <= bound
    m = 60                                                          # a further piece of both rows
    q2, k2, v2 = mk(hq, m), mk(H, m), mk(H, m)
    rq2 = kb.kv8_append(layer, k2, v2, n, rotary=rot, query=q2)
    n2 = n + m
    ke, ve = kb.kv8_expand(layer, n2, L + 3 + m)
    piece = kb.prompt_attention(rq2, ke, ve, SC, key_lengths=n2)
    for b in range(B):
        w = int(n2[b])
        lim = torch.arange(m, device=DEV) + 1 + w - m
        for x in range(hq):
            a, kk, vv = rq2[b, x].double(), ke[b, x // 4, :w].double(), ve[b, x // 4, :w].double()
            want, mag = attend_fast(a, kk, vv, SC, lim)
            assert ((piece[b, :, x].double() - want).abs()
                    <= attention_bound(want, mag, dtype, HALF[dtype], logit_error(a, kk, SC))).all()
    assert torch.isfinite(prompt).all() and (prompt[1, 77:] == 0).all()
    layer.check()
    assert kb.prompt_attention_status(DEV) == 0


def test_rows_off_their_boundaries(kb):
    k, v = _kv(1, 2, 40, torch.float16, 4)
    wide = torch.zeros(1, 2, 40, 130, dtype=torch.float16, device=DEV)
    wide[..., 1:129] = k
    a, b = (kb.KV8Layer(1, 128, 2, dtype=torch.float16, device=DEV) for _ in range(2))
    kb.kv8_append(a, k, v, _i32([0]))
    kb.kv8_append(b, wide[..., 1:129], v, _i32([0]))
    assert torch.equal(a.pages, b.pages) and torch.equal(a.tail_k, b.tail_k)


def test_a_replaced_page_table_is_used_and_checked(kb):
    k, v = _kv(1, 1, 128, torch.bfloat16, 5)
    layer = kb.KV8Layer(1, 256, 1, device=DEV)
    kb.kv8_append(layer, k, v, _i32([0]))
    first = layer.pages[0].clone()
    layer.page_table = torch.tensor([[1, 0]], device=DEV)
    kb.kv8_append(layer, k, v, _i32([0]))
    assert torch.equal(layer.pages[1], first)
    layer.page_table = torch.zeros(1, 3, dtype=torch.int64, device=DEV)
    with pytest.raises(ValueError, match="page_table"):
        kb.kv8_append(layer, k, v, _i32([0]))


def test_tensors_that_want_a_gradient_are_refused(kb):
    lay = kb.KV8Layer(1, 128, 1, device=DEV)
    rot, z = kb.RotaryEmbedding(device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    x, g = (torch.randn(1, 1, 1, 128, device=DEV).bfloat16().requires_grad_(want) for want in (False, True))
    pos = torch.zeros(1, dtype=torch.int64, device=DEV)
    calls = [lambda: kb.kv8_append(lay, g, x, z), lambda: kb.kv8_append(lay, x, g, z),
             lambda: kb.kv8_append(lay, x, x, z, rotary=rot, query=g), lambda: kb.kv8_attention(g, lay, z, 1.0),
             lambda: kb.apply_rotary(g, x, pos, rot), lambda: kb.apply_rotary(x, g, pos, rot)]
    for call in calls:
        with pytest.raises(ValueError, match="no backward pass"):
            call()
        with torch.no_grad():
            call()
    lay.check()


@pytest.mark.parametrize("room", [0, 4100])
@pytest.mark.parametrize("scaling", [0.0, -0.3, 1e-30, 3.0])
def test_scalings_of_any_sign_and_size(kb, scaling, room):
    """Zero is the mean of the values, a negative one turns the order around, a large one picks a few tokens."""
    lengths = [333, 0, 45]
    layer = kb.KV8Layer(3, 333 + room, 2, device=DEV)
    k, v = _kv(3, 2, 333, torch.bfloat16, 9)
    n = _i32(lengths)
    kb.kv8_append(layer, k, v, torch.zeros_like(n), lengths=n)
    q = torch.randn(3, 6, 1, 128, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).bfloat16()
    _attention_check(kb.kv8_attention(q, layer, n, scaling), q, layer, lengths, (k, v), scaling)
    layer.check()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,H,cap,lengths", [
    (3, 1, 640, [128, 512, 600]),                       # a block of threads per row
    (150, 1, 640, [128, 512, 600] + [96] * 147),        # four warps a row
    (3, 2, 4096, [128, 2048, 3900]),                    # split over workers, joined by blocks
    (130, 2, 9000, [128, 2048, 8900] + [96] * 127)])    # joined by warps; short rows that one worker has whole
@pytest.mark.parametrize("hq_per", [1, 12])
def test_rows_whose_pages_are_all_bad(kb, dtype, B, H, cap, lengths, hq_per):
    """Blocks of bad pages count as not held: a row that keeps nothing is zero, one that keeps its open block is that."""
    pages = -(-cap // 128)
    layer = kb.KV8Layer(B, cap, H, dtype=dtype, device=DEV, num_pages=200, page_table=torch.full((B, pages), -7, device=DEV))
    k, v = _kv(B, H, max(lengths) + 5, dtype, 31)
    g = torch.Generator(device=DEV).manual_seed(32)
    q = torch.randn(B, H * hq_per, 1, 128, generator=g, device=DEV).to(dtype)
    n = _i32(lengths)
    kb.kv8_append(layer, k, v, torch.zeros_like(n), lengths=n)             # open blocks only: the pages are bad
    got = kb.kv8_attention(q, layer, n, SC)
    for b, m in enumerate(lengths):
        full = m // 32 * 32
        if m == full:
            assert (got[b] == 0).all(), b
            continue
        for x in range(H * hq_per):
            want, mag = attend_fast(q[b, x].double(), k[b, x // hq_per, full:m].double(), v[b, x // hq_per, full:m].double(), SC,
                                    torch.tensor([m - full], device=DEV))
            bound = attention_bound(want, mag, dtype, 2.0 ** -16, logit_error(q[b, x].double(), k[b, x // hq_per, full:m].double(), SC))
            assert ((got[b, :, x].double() - want).abs() <= bound).all(), (b, x)
    with pytest.raises(ValueError, match="page-table"):
        layer.check()


@pytest.mark.parametrize("room", [0, 4100])
def test_logits_that_are_all_minus_infinity(kb, room):
    """Not the same as a row without tokens: zero over zero."""
    layer = kb.KV8Layer(1, 100 + room, 1, dtype=torch.float16, device=DEV)
    k, v = torch.zeros(1, 1, 7, 128, device=DEV).half(), torch.ones(1, 1, 7, 128, device=DEV).half()
    k[..., 5] = float("-inf")
    kb.kv8_append(layer, k, v, _i32([0]))
    q = torch.zeros(1, 2, 1, 128, device=DEV).half()
    q[..., 5] = 1.0
    assert torch.isnan(kb.kv8_attention(q, layer, _i32([7]), SC)).all()
    layer.check()


@pytest.mark.parametrize("B,cap,lengths", [(2, 640, [600, 77]), (150, 640, [33, 600] + [96] * 148), (2, 4096, [3900, 100]),
                                           (300, 9000, [600, 40] + [96] * 298)])
def test_output_in_the_query_s_own_place(kb, B, cap, lengths):
    """Row for row over the query, on each of the ways a call can take."""
    layer = kb.KV8Layer(B, cap, 1, device=DEV, num_pages=1000,
                        page_table=(torch.arange(B * -(-cap // 128), device=DEV) % 1000).view(B, -1))
    k, v = _kv(B, 1, 600, torch.bfloat16, 41)
    n = _i32(lengths)
    kb.kv8_append(layer, k, v, torch.zeros_like(n), lengths=n.clamp(max=600))
    q = torch.randn(B, 6, 1, 128, generator=torch.Generator(device=DEV).manual_seed(42), device=DEV).bfloat16()
    want = kb.kv8_attention(q, layer, n, SC)
    for _ in range(5):
        mine = q.clone()
        got = kb.kv8_attention(mine, layer, n, SC, out=mine.view(B, 1, 6, 128))
        assert got.data_ptr() == mine.data_ptr() and torch.equal(got, want)
    buf = torch.zeros(B + 1, 6, 128, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="overlaps"):
        kb.kv8_attention(buf[:B].view(B, 6, 1, 128), layer, n, SC, out=buf[1:].view(B, 1, 6, 128))


@pytest.mark.parametrize("rotated", [False, True])
def test_what_refused_and_clamped_appends_store(kb, rotated):
    """A count below zero or a start outside stores nothing; too many tokens are stored as far as they go.  Other rows of the
    call are stored as ever."""
    T, cap = 40, 256
    rot = kb.RotaryEmbedding(device=DEV) if rotated else None
    k, v = _kv(2, 2, T, torch.bfloat16, 51)
    k0, v0 = _kv(2, 2, 250, torch.bfloat16, 52)

    def held(start, n):
        layer = kb.KV8Layer(2, cap, 2, device=DEV)
        kb.kv8_append(layer, k0, v0, _i32([0, 0]))                          # 250 tokens each: 26 in the open block
        if n is not None:
            kb.kv8_append(layer, k, v, _i32(start), lengths=None if n == "all" else _i32(n), rotary=rot)
        return layer

    same = lambda a, b, row: all(torch.equal(getattr(a, x).view(2, -1)[row], getattr(b, x).view(2, -1)[row])  # noqa: E731
                                 for x in ("pages", "tail_k", "tail_v"))
    before = held(None, None)
    for start, n, row in (([250, 250], [-3, 5], 0), ([-1, 250], [5, 5], 0), ([257, 250], [5, 5], 0), ([250, 1 << 30], [5, 5], 1),
                          ([250, -(1 << 31)], [5, 5], 1), ([250, 250], [5, -(1 << 31)], 1)):
        got = held(start, n)
        want = held([250, 250], [0, 5] if row == 0 else [5, 0])
        assert same(got, before, row) and same(got, want, 1 - row), (start, n)
        with pytest.raises(ValueError, match="length"):
            got.check()
    # six of the tokens fit; more than the call has are what it has
    fits = held([250, 250], [6, 6])
    fits.check()
    for n in ("all", [40, 6], [7, 1 << 30]):
        got = held([250, 250], n)
        assert same(got, fits, 0) and same(got, fits, 1)
        with pytest.raises(ValueError, match="length"):
            got.check()
    got, want = held([100, 256], [999, 3]), held([100, 256], [40, 0])       # a full row takes nothing
    assert same(got, want, 0) and same(got, before, 1)
    with pytest.raises(ValueError, match="length"):
        got.check()


def test_the_last_tokens_of_the_longest_cache(kb):
    """Positions up to 2^30, in calls of up to 2^30 tokens: block numbers whose tokens pass 2^31."""
    cap = 1 << 30
    layer = kb.KV8Layer(1, cap, 1, device=DEV, num_pages=2, page_table=torch.zeros(1, cap // 128, dtype=torch.int64, device=DEV))
    layer.page_table[0, -1] = 1
    k, v = _kv(1, 1, 64, torch.bfloat16, 61)
    one = kb.KV8Layer(1, 64, 1, device=DEV)
    kb.kv8_append(one, k, v, _i32([0]))
    kb.kv8_append(layer, k, v, _i32([cap - 64]))
    layer.check()
    assert torch.equal(layer.pages[1, :, 2:], one.pages[0, :, :2]) and (layer.pages[0] == 0).all()
    # the most tokens that a call may have (all of them the same one): those that still fit are stored
    many = (x[:, :, :1].expand(1, 1, cap, 128) for x in (k, v))
    kb.kv8_append(layer, *many, _i32([cap - 32]))
    with pytest.raises(ValueError, match="length"):
        layer.check()
    same = kb.KV8Layer(1, 32, 1, device=DEV)
    kb.kv8_append(same, k[:, :, :1].expand(1, 1, 32, 128), v[:, :, :1].expand(1, 1, 32, 128), _i32([0]))
    assert torch.equal(layer.pages[1, :, 3], same.pages[0, :, 0]) and torch.equal(layer.pages[1, :, 2], one.pages[0, :, 0])
    assert (layer.pages[0] == 0).all() and (layer.pages[1, :, :2] == 0).all()
    ke, ve = kb.kv8_expand(layer, _i32([cap]), 70, start=_i32([cap - 50]))
    assert torch.equal(ke[0, :, :18], _held(k[0], 32, torch.bfloat16)[:, 14:]) and (ke[0, :, 50:] == 0).all()
    assert torch.equal(ve[0, :, 18:50], _held(v[0, :, :1].expand(1, 32, 128), 32, torch.bfloat16))


def test_autograd_notices_lent_outputs(kb):
    """A tensor saved for a backward pass and then lent as an output: that backward pass says so."""
    x = lambda *s: torch.randn(*s, device=DEV).bfloat16()                   # noqa: E731
    w = torch.ones(1, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    rot, pos = kb.RotaryEmbedding(device=DEV), torch.arange(3, device=DEV)
    layer, n = kb.KV8Layer(1, 128, 1, device=DEV), _i32([3])
    kb.kv8_append(layer, x(1, 1, 3, 128), x(1, 1, 3, 128), _i32([0]))
    q, k, v, o = x(1, 2, 3, 128), x(1, 1, 3, 128), x(1, 1, 3, 128), x(1, 3, 2, 128)
    o1 = x(1, 1, 2, 128)
    for saved, call in ((q, lambda: kb.apply_rotary(q, k, pos, rot, query_out=q, key_out=k)),
                        (k, lambda: kb.apply_rotary(q, k, pos, rot, key_out=k)),
                        (o, lambda: kb.prompt_attention(q, k, v, SC, out=o)),
                        (o1, lambda: kb.kv8_attention(q[:, :, :1], layer, n, SC, out=o1))):
        y = (w * saved).sum()
        call()
        with pytest.raises(RuntimeError, match="inplace"):
            y.backward()
    with torch.inference_mode():                                            # and inference tensors are lent as ever
        q = x(1, 2, 3, 128)
        kb.apply_rotary(q, k, pos, rot, query_out=q)
    kb.apply_rotary(q, k, pos, rot, query_out=q)
    y = (w * k).sum()
    kb.apply_rotary(q, k, pos, rot)                                         # nothing lent, nothing written
    y.backward()


@pytest.mark.parametrize("dtype,hq", [(torch.bfloat16, 4), (torch.float16, 7), (torch.bfloat16, 16)])
def test_attention_long_rows(kb, dtype, hq):
    """Rows of up to 70000 tokens beside short ones: many partials of one row, and workers that end within rows."""
    lengths = [70001, 31, 40000, 0, 517]
    B, pages = len(lengths), [-(-n // 128) for n in lengths]
    table = torch.zeros(B, max(pages), dtype=torch.int64)
    at = 0
    order = torch.randperm(sum(pages), generator=torch.Generator().manual_seed(71))
    for b, m in enumerate(pages):
        table[b, :m] = order[at:at + m]
        at += m
    layer = kb.KV8Layer(B, max(lengths), 1, dtype=dtype, device=DEV, num_pages=at, page_table=table.to(DEV))
    k, v = _kv(B, 1, max(lengths), dtype, 72)
    n = _i32(lengths)
    kb.kv8_append(layer, k, v, torch.zeros_like(n), lengths=n)
    q = torch.randn(B, hq, 1, 128, generator=torch.Generator(device=DEV).manual_seed(73), device=DEV).to(dtype)
    got = kb.kv8_attention(q, layer, n, SC)
    _attention_check(got, q, layer, lengths, (k, v), SC)
    assert torch.equal(kb.kv8_attention(q, layer, n, SC), got)
    layer.check()


@pytest.mark.parametrize("room", [0, 4100])
@pytest.mark.parametrize("size", [30.0, 1000.0])
def test_a_query_channel_far_above_the_others(kb, room, size):
    """The other channels keep 1/65024 of it, as the bound says."""
    lengths = [700, 90]
    layer = kb.KV8Layer(2, 700 + room, 2, device=DEV)
    k, v = _kv(2, 2, 700, torch.bfloat16, 81)
    n = _i32(lengths)
    kb.kv8_append(layer, k, v, torch.zeros_like(n), lengths=n)
    q = torch.randn(2, 6, 1, 128, generator=torch.Generator(device=DEV).manual_seed(82), device=DEV)
    q[..., 77] *= size
    q = q.bfloat16()
    _attention_check(kb.kv8_attention(q, layer, n, SC), q, layer, lengths, (k, v), SC)
    layer.check()


def test_append_turns_a_query_in_place(kb):
    """The entry point's rotated query may be the query itself."""
    from kitty_b200 import _lib

    rot = kb.RotaryEmbedding(rotary_dim=96, device=DEV)
    k, v = _kv(2, 2, 70, torch.bfloat16, 91)
    q = torch.randn(2, 6, 70, 128, generator=torch.Generator(device=DEV).manual_seed(92), device=DEV).bfloat16()
    a, b = (kb.KV8Layer(2, 128, 2, device=DEV) for _ in range(2))
    start = _i32([0, 5])
    want = kb.kv8_append(a, k, v, start, rotary=rot, query=q)
    st = [_lib.head_rows(x)[1] for x in (k, v, q)]
    _lib.call_on(b.device, _lib.lib().kitty_kv8_append, "kitty_kv8_append", b.c_layer(), k.data_ptr(), v.data_ptr(),
                 _lib.i64_array(st[0] + st[1] + st[2]), start.data_ptr(), None, 2, 70, rot.c_plan(), q.data_ptr(), q.data_ptr(), 6)
    assert torch.equal(q, want) and torch.equal(a.pages, b.pages)
