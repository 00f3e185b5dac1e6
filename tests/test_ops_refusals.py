"""What the prompt-side operators and the 8-bit cache refuse (no GPU needed: every check comes before the first launch)."""
import ctypes as C
import math

import pytest
import torch

P = 4096            # stands for an aligned pointer: refused calls never follow it


@pytest.fixture(scope="module")
def L():
    from kitty_b200 import _lib

    return _lib


def _plan(L, r=128, layout=0, turns=P):
    return L.KittyRotaryPlan(turns, P, 1.0, r, layout, 0)


def _layer(L, **over):
    f = dict(max_bs=4, max_page=8, num_pages=32, h_kv=2, head_dim=128, dtype=L.KITTY_BF16, pages=P, tail_k=P, tail_v=P,
             page_table=P, status=P)
    f.update(over)
    return L.KittyKV8Layer(*f.values())


def _rotary(L, plan, q=P, k=P, pos=P, pos_b=0, qo=P, ko=P, dtype=0, B=1, T=1, hq=1, h=1, st=(0,) * 12):
    return L.lib().kitty_rotary(plan, q, k, pos, pos_b, qo, ko, dtype, B, T, hq, h, L.i64_array(list(st)), None)


def test_rotary_entry_point(L):
    assert _rotary(L, None) == L.KITTY_E_BADARG
    assert _rotary(L, _plan(L, turns=None)) == L.KITTY_E_BADARG
    for r in (0, 3, 130, -2):
        assert _rotary(L, _plan(L, r)) == L.KITTY_E_BADSHAPE
    assert _rotary(L, _plan(L, layout=2)) == L.KITTY_E_BADARG
    good = _plan(L)
    for kw in (dict(q=None), dict(k=None), dict(pos=None), dict(qo=None), dict(dtype=3), dict(B=-1), dict(T=-1), dict(q=P + 2),
               dict(ko=P + 8), dict(hq=-1), dict(pos_b=-1), dict(st=(4,) + (0,) * 11), dict(dtype=2, st=(2,) + (0,) * 11)):
        assert _rotary(L, good, **kw) == L.KITTY_E_BADARG, kw
    assert _rotary(L, good, B=0) == L.KITTY_OK and _rotary(L, good, T=0, q=None, k=None) == L.KITTY_OK


def _prompt(L, q=P, k=P, v=P, dtype=0, st=(0,) * 9, B=1, Lq=1, Lk=1, hq=1, h=1, sc=1.0, ql=None, kl=None, cu=None, cuk=None,
            out=P, ws=None, nbytes=0):
    return L.lib().kitty_prompt_attn(q, k, v, dtype, L.i64_array(list(st)), B, Lq, Lk, hq, h, sc, 1, ql, kl, cu, cuk, out, 0,
                                     None, ws, nbytes, None)


def test_prompt_entry_point(L):
    for kw in (dict(q=None), dict(k=None), dict(out=None), dict(dtype=2), dict(dtype=7), dict(hq=3, h=2), dict(h=0), dict(hq=0),
               dict(B=-1), dict(Lq=-1), dict(sc=0.0), dict(sc=-1.0), dict(sc=math.inf), dict(sc=math.nan), dict(q=P + 8),
               dict(out=P + 4), dict(Lq=2), dict(Lq=2, st=(0, 0, 4) + (0,) * 6), dict(Lk=2, st=(0,) * 5 + (-128,) + (0,) * 3)):
        assert _prompt(L, **kw) == L.KITTY_E_BADARG, kw
    assert _prompt(L, Lq=(1 << 30) + 1) == L.KITTY_E_BADSHAPE
    need = L.lib().kitty_prompt_workspace_bytes
    assert need(1, 1, 100000, 8, 1, 1, 0) > 0 and need(16, 4096, 4096, 32, 8, 1, 0) == 0 and need(0, 0, 0, 1, 1, 1, 1) == 0
    assert need(1, 1, 1, 3, 2, 1, 0) == L.KITTY_E_BADARG and need(1, 1 << 31, 1, 1, 1, 1, 0) == L.KITTY_E_BADSHAPE
    far = dict(Lk=100000, hq=8, h=1, st=(0, 128, 0) + (0, 0, 128) * 2)
    assert _prompt(L, ws=P, nbytes=16, **far) == L.KITTY_E_WORKSPACE
    assert _prompt(L, ws=P + 8, nbytes=1 << 40, **far) == L.KITTY_E_BADARG
    assert _prompt(L, B=0) == L.KITTY_OK and _prompt(L, Lq=0) == L.KITTY_OK


def test_kv8_entry_points(L):
    lib = L.lib()
    z9 = L.i64_array([0] * 9)

    def append(layer, k=P, v=P, st=z9, start=P, B=1, T=1, plan=None, q=None, qo=None, hq=0):
        return lib.kitty_kv8_append(layer, k, v, st, start, None, B, T, plan, q, qo, hq, None)

    def expand(layer, n=4, lens=P, k=P, v=P, B=1):
        return lib.kitty_kv8_expand(layer, lens, None, k, v, B, n, None)

    def attn(layer, lens=P, q=P, B=1, hq=2, out=P, ws=P, nbytes=1 << 40):
        return lib.kitty_kv8_attn(layer, lens, q, B, hq, 1.0, out, ws, nbytes, None)

    for over in (dict(pages=None), dict(tail_k=None), dict(page_table=None), dict(status=None), dict(dtype=2), dict(max_bs=0),
                 dict(num_pages=0), dict(h_kv=0), dict(max_page=-1), dict(pages=P + 8)):
        bad = _layer(L, **over)
        assert append(bad) == expand(bad) == attn(bad) == L.KITTY_E_BADARG, over
    for over in (dict(head_dim=64), dict(max_page=(1 << 23) + 1)):
        bad = _layer(L, **over)
        assert append(bad) == expand(bad) == attn(bad) == L.KITTY_E_BADSHAPE, over
    good = _layer(L)
    for kw in (dict(k=None), dict(v=P + 2), dict(start=None), dict(B=5), dict(B=-1), dict(T=-1), dict(hq=2, q=P, qo=P),
               dict(hq=2, plan=_plan(L), q=None, qo=P), dict(hq=2, plan=_plan(L), q=P, qo=None), dict(plan=_plan(L, layout=5)),
               dict(st=L.i64_array([4] + [0] * 8)), dict(hq=1, plan=_plan(L), q=P, qo=P, st=L.i64_array([0] * 8 + [2]))):
        assert append(good, **kw) == L.KITTY_E_BADARG, kw
    assert append(good, T=0) == append(good, B=0) == L.KITTY_OK
    for kw in (dict(lens=None), dict(k=None), dict(v=P + 8), dict(B=5), dict(n=-1)):
        assert expand(good, **kw) == L.KITTY_E_BADARG, kw
    assert expand(good, n=0) == L.KITTY_OK
    for kw in (dict(lens=None), dict(q=None), dict(q=P + 4), dict(out=None), dict(B=5), dict(hq=3), dict(hq=0)):
        assert attn(good, **kw) == L.KITTY_E_BADARG, kw
    assert attn(good, hq=34) == L.KITTY_E_BADSHAPE
    assert attn(_layer(L, max_page=64), nbytes=100) == L.KITTY_E_WORKSPACE
    assert attn(_layer(L, max_page=64), ws=None) == L.KITTY_E_BADARG
    assert attn(good, B=0) == L.KITTY_OK
    need = lib.kitty_kv8_workspace_bytes
    assert need(1, 2, 3, 64) == need(1, 2, 4, 0) == L.KITTY_E_BADARG
    assert need(L.KV8_MAX_BATCH + 1, 2, 4, 64) == L.KITTY_E_BADSHAPE
    assert need(128, 8, 32, 64) > need(1, 8, 32, 64) > 0 and need(1, 8, 32, 8) == need(32, 8, 32, 32) == 0


def test_struct_sizes(L):
    assert C.sizeof(L.KittyRotaryPlan) == 32 and C.sizeof(L.KittyKV8Layer) == 6 * 4 + 5 * 8


def test_python_refusals_without_a_gpu():
    import kitty_b200 as kb
    from kitty_b200.rotary import _scaled_frequencies

    x = torch.zeros(1, 2, 4, 128, dtype=torch.float16)
    for bad in (dict(head_dim=64), dict(rotary_dim=3), dict(rotary_dim=130), dict(layout="pairs"), dict(base=0.0),
                dict(base=math.inf), dict(device="cpu"), dict(scaling={"rope_type": "dynamic", "factor": 2.0}),
                dict(scaling={"rope_type": "linear", "factor": -1.0}),
                dict(scaling={"rope_type": "yarn", "factor": 2.0, "original_max_position_embeddings": 0}),
                dict(scaling={"rope_type": "yarn", "factor": 2.0, "original_max_position_embeddings": 4096, "mscale": 1.0}),
                dict(scaling={"rope_type": "llama3", "factor": 2.0, "original_max_position_embeddings": 4096,
                              "low_freq_factor": 4.0, "high_freq_factor": 4.0})):
        with pytest.raises(ValueError):
            kb.RotaryEmbedding(**{"device": "cpu", **bad})
    import types

    with pytest.raises(ValueError, match="CUDA"):
        kb.apply_rotary(x, x, torch.arange(4), types.SimpleNamespace(device=torch.device("cuda", 0)))
    with pytest.raises(ValueError, match="CUDA"):
        kb.prompt_attention(x, x, x, 1.0)
    with pytest.raises(ValueError, match="expected query"):
        kb.prompt_attention(x[0], x, x, 1.0)
    for bad in (dict(MAX_BS=0), dict(MAX_LEN=0), dict(H_KV=0), dict(D=64), dict(MAX_LEN=(1 << 30) + 1), dict(device="cpu")):
        with pytest.raises(ValueError):
            kb.KV8Layer(**{**dict(MAX_BS=1, MAX_LEN=128, H_KV=1, device="cpu"), **bad})
    with pytest.raises(TypeError):
        kb.KV8Layer(1, 128, 1, dtype=torch.float32, device="cpu")
    assert _scaled_frequencies(4, 10000.0, {"rope_type": "default"}) == ([1.0, 0.01], 1.0)


def test_scaled_frequencies_match_transformers():
    """The angles of the scalings are those of transformers' own configurations (which it keeps in 32 bits)."""
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

    from kitty_b200.rotary import _scaled_frequencies

    for scaling in ({"rope_type": "linear", "factor": 4.0},
                    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                     "original_max_position_embeddings": 8192},
                    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}):
        for base in (10000.0, 500000.0):
            cfg = LlamaConfig(hidden_size=512, num_attention_heads=4, max_position_embeddings=131072,
                              rope_parameters={**scaling, "rope_theta": base})
            want, factor = ROPE_INIT_FUNCTIONS[scaling["rope_type"]](cfg, torch.device("cpu"))
            inv, f = _scaled_frequencies(128, base, scaling)
            got = torch.tensor(inv, dtype=torch.float64)
            assert ((got - want.double()).abs() <= 2.0 ** -20 * got).all() and abs(f - factor) < 1e-12


def test_gradients_are_refused(L):
    import kitty_b200 as kb

    x = torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16)
    for i in range(3):
        a = [x.clone().requires_grad_(j == i) for j in range(3)]
        with pytest.raises(ValueError, match="no backward pass"):
            kb.prompt_attention(*a, 1.0)
        with torch.no_grad(), pytest.raises(ValueError, match="no CPU path"):
            kb.prompt_attention(*a, 1.0)
    L.refuse_gradients("it", x)
    with pytest.raises(ValueError, match="it has no backward pass"):
        L.refuse_gradients("it", x, x.clone().requires_grad_())


def _meet(L, x, y, run):
    """x, y: (address, sizes, steps in bytes)."""
    (a, n, s), (b, m, t) = x, y
    return bool(L.lib().kitty_rows_overlap(a, L.i64_array(n), L.i64_array(s), b, L.i64_array(m), L.i64_array(t), run))


def test_whether_rows_share_memory(L):
    """Against the sets of bytes themselves: nested and fused layouts, expanded dimensions, steps that do not nest."""
    import random

    rng = random.Random(5)

    def bytes_of(at, n, s, run):
        out = {at}
        for size, step in zip(n, s):
            out = {x + i * step for x in out for i in range(size)}
        return {x + i for x in out for i in range(run)}

    met = apart = 0
    for _ in range(4000):
        run = rng.choice([2, 4])
        n = [[rng.choice([1, 1, 2, 3]) for _ in range(3)] for _ in range(2)]
        if rng.random() < 0.6:                       # both from one buffer, as slices of a fused projection are
            st, step = [], run
            for _ in range(3):
                st.append(step)
                step *= rng.choice([2, 3, 4])
            rng.shuffle(st)
            s = [st, st]
        else:
            s = [[run * rng.randrange(-3, 9) for _ in range(3)] for _ in range(2)]
        at = 1000 + rng.randrange(-12, 13) * rng.choice([1, run])
        want = bool(bytes_of(1000, n[0], s[0], run) & bytes_of(at, n[1], s[1], run))
        assert _meet(L, (1000, n[0], s[0]), (at, n[1], s[1]), run) == want, (n, s, at, run)
        met, apart = met + want, apart + (not want)
    assert met > 500 and apart > 500
    assert not _meet(L, (1000, (0, 2, 1), (4, 8, 16)), (1000, (2, 2, 1), (4, 8, 16)), 4)
    # rows of 256 bytes, [2, T, 40, 128] in 16 bits: 32 query and 8 key heads of one buffer; the same at 2^31 rows
    for T in (4096, 1 << 30):
        st = (T * 10240, 256, 10240)
        q, k = (1 << 20, (2, 32, T), st), ((1 << 20) + 32 * 256, (2, 8, T), st)
        assert not _meet(L, q, k, 256) and not _meet(L, k, q, 256) and _meet(L, q, (q[0] + 31 * 256, (2, 8, T), st), 256)
        assert _meet(L, q, (k[0] + 8 * 256, (2, 8, T), st), 256) and not _meet(L, q, (q[0] + 2 * T * 10240, (1, 1, 1), (0, 0, 0)), 256)


def test_outputs_that_share_memory_are_refused(L):
    """Refused before anything is launched, whatever else the call holds."""
    H = 256                                           # bytes of a 16-bit row
    fused = (5 * 12 * 128, 128, 12 * 128)             # [B, T, 12 heads, 128]: heads 0-3 query, 4-7 key, 8-11 others
    rot = lambda qo, ko: _rotary(L, _plan(L), q=P, k=P + 4 * H, qo=P + qo * H, ko=P + ko * H, B=2, T=5, hq=4, h=4,  # noqa: E731
                                 st=fused * 4)
    for qo, ko in ((4, 0), (4, 8), (8, 0), (8, 8), (1, 8), (8, 5), (0, 0), (8, 9), (0, 3)):
        assert rot(qo, ko) == L.KITTY_E_OVERLAP, (qo, ko)
    # the same place, but in another order
    assert _rotary(L, _plan(L), q=P, k=1 << 30, qo=P, ko=1 << 30, B=1, T=5, hq=4, h=4, st=(0, 128, 512) + (0, 640, 128) * 3) \
        == L.KITTY_E_OVERLAP
    heads = (7 * 4 * 128, 128, 4 * 128)
    far = 1 << 30
    one = dict(B=2, Lq=7, Lk=7, hq=4, h=4, out=P)
    for where in "qkv":
        at = dict(q=far, k=2 * far, v=3 * far)
        for shift in (0, 3 * H, -2 * 7 * 4 * H + H):
            assert _prompt(L, **{**at, where: P + far + shift}, **{**one, "out": P + far}, st=heads * 3) == L.KITTY_E_OVERLAP
    assert _prompt(L, q=P, k=far, v=2 * far, **one, st=(7 * 4 * 128, 7 * 128, 128) + heads * 2) == L.KITTY_E_OVERLAP
    assert _prompt(L, q=P, k=far, v=2 * far, cu=P, **{**one, "B": 1}, st=(0, 128, 512) * 3) == L.KITTY_E_OVERLAP
    lib, layer = L.lib(), _layer(L, h_kv=2)
    for shift in (H, -H, 3 * H):
        assert lib.kitty_kv8_attn(layer, P, far, 2, 2, 1.0, far + shift, P, 1 << 40, None) == L.KITTY_E_OVERLAP
    assert lib.kitty_kv8_expand(layer, P, None, far, far + 5 * H, 2, 4, None) == L.KITTY_E_OVERLAP
    st = L.i64_array((2 * 6 * 128, 6 * 128, 128) * 2 + (2 * 6 * 128, 128, 2 * 128))
    assert lib.kitty_kv8_append(layer, far, 2 * far, st, P, None, 2, 6, _plan(L), 3 * far, 3 * far, 2, None) == L.KITTY_E_OVERLAP
    st = L.i64_array((2 * 6 * 128, 6 * 128, 128) * 3)
    for name in ("key", "value", "query"):
        at = {"key": far, "value": 2 * far, "query": 3 * far}
        assert lib.kitty_kv8_append(layer, at["key"], at["value"], st, P, None, 2, 6, _plan(L), at["query"], at[name] + 3 * H, 2,
                                    None) == L.KITTY_E_OVERLAP
    assert "overlaps" in L.strerror(L.KITTY_E_OVERLAP)


def _angles(monkeypatch, **kw):
    """What a RotaryEmbedding makes of its arguments before it goes to a device: (rotary_dim, base, scaling)."""
    import kitty_b200 as kb
    from kitty_b200 import rotary

    seen = []
    real = rotary._scaled_frequencies
    monkeypatch.setattr(rotary, "_scaled_frequencies", lambda *a: seen.append(a) or real(*a))
    with pytest.raises(ValueError, match="no CPU path"):
        kb.RotaryEmbedding(device="cpu", **kw)
    return seen[0]


def test_rope_parameters_are_taken_or_refused(monkeypatch):
    """rope_theta and partial_rotary_factor come with a configuration's rope parameters: honoured, and refused where an
    argument says otherwise."""
    from transformers import LlamaConfig

    import kitty_b200 as kb

    cfg = LlamaConfig(rope_parameters={"rope_type": "llama3", "rope_theta": 500000.0, "factor": 8.0, "low_freq_factor": 1.0,
                                       "high_freq_factor": 4.0, "original_max_position_embeddings": 8192})
    assert _angles(monkeypatch, scaling=cfg.rope_parameters)[:2] == (128, 500000.0)
    assert _angles(monkeypatch, scaling=cfg.rope_parameters, base=500000.0, rotary_dim=64)[:2] == (64, 500000.0)
    assert _angles(monkeypatch, scaling={"rope_type": "default", "rope_theta": 1000000})[:2] == (128, 1000000.0)
    half = {"rope_type": "linear", "factor": 2.0, "rope_theta": 10000.0, "partial_rotary_factor": 0.5}
    assert _angles(monkeypatch, scaling=half)[:2] == (64, 10000.0) and _angles(monkeypatch, scaling=half, rotary_dim=64)[0] == 64
    assert _angles(monkeypatch)[:2] == (128, 10000.0) and _angles(monkeypatch, base=5.0)[:2] == (128, 5.0)
    for bad, what in ((dict(base=10000.0, scaling=cfg.rope_parameters), "rope_theta"), (dict(rotary_dim=128, scaling=half), "partial_rotary_factor"),
                      (dict(scaling={"rope_theta": 0.0}), "base must be"), (dict(scaling={**half, "partial_rotary_factor": 0.4}), "rotary_dim")):
        with pytest.raises(ValueError, match=what):
            kb.RotaryEmbedding(device="cpu", **bad)


def test_scalings_are_refused_by_name():
    """Each for its own reason."""
    from kitty_b200.rotary import _scaled_frequencies

    llama3 = {"rope_type": "llama3", "factor": 2.0, "original_max_position_embeddings": 4096, "low_freq_factor": 1.0, "high_freq_factor": 4.0}
    yarn = {"rope_type": "yarn", "factor": 2.0, "original_max_position_embeddings": 4096}
    linear = {"rope_type": "linear", "factor": 2.0}
    for scaling in (llama3, yarn, linear, {"rope_type": "default"}, {"type": "linear", "factor": 3}, {}):
        assert len(_scaled_frequencies(128, 10000.0, scaling)[0]) == 64
    for scaling, what in (({"rope_type": "dynamic", "factor": 2.0}, "'dynamic' is not supported"), ({"rope_type": None}, "None is not supported"),
                          ({**linear, "factor": -1.0}, "factor must be positive"), ({**linear, "factor": math.inf}, "factor must be positive"),
                          ({"rope_type": "linear"}, "needs factor"), ({**linear, "low_freq_factor": 1.0}, "with low_freq_factor"),
                          ({"rope_type": "default", "mrope_section": [1]}, "with mrope_section"),
                          ({"full_attention": linear}, "with full_attention"),
                          ({**llama3, "high_freq_factor": 1.0}, "high_freq_factor must be above"), ({**llama3, "beta_fast": 3}, "with beta_fast"),
                          ({k: v for k, v in llama3.items() if k[:4] != "low_"}, "needs low_freq_factor"),
                          ({**llama3, "original_max_position_embeddings": None}, "needs original_max"),
                          ({**yarn, "original_max_position_embeddings": 0}, "original_max_position_embeddings must be positive"),
                          ({**yarn, "mscale": 1.0}, "with mscale"), ({**yarn, "factor": None}, "needs factor")):
        with pytest.raises(ValueError, match=what):
            _scaled_frequencies(128, 10000.0, scaling)
    with pytest.raises(ValueError, match="base other than 1"):
        _scaled_frequencies(128, 1.0, yarn)


def test_constructors_refuse_each_for_its_own_reason():
    import kitty_b200 as kb

    for bad, what in ((dict(head_dim=64), "head_dim=128"), (dict(rotary_dim=3), "rotary_dim must be even"), (dict(rotary_dim=130), "rotary_dim"),
                      (dict(rotary_dim=0), "rotary_dim"), (dict(layout="pairs"), "layout must be"), (dict(base=0.0), "base must be positive"),
                      (dict(base=math.inf), "base must be positive"), (dict(base=math.nan), "base must be positive"), ({}, "no CPU path")):
        with pytest.raises(ValueError, match=what):
            kb.RotaryEmbedding(**{"device": "cpu", **bad})
    for bad, what in ((dict(MAX_BS=0), "must be positive"), (dict(MAX_LEN=0), "must be positive"), (dict(H_KV=-1), "must be positive"),
                      (dict(D=64), "D=128"), (dict(MAX_LEN=(1 << 30) + 1), "2\\^30"), ({}, "no CPU path")):
        with pytest.raises(ValueError, match=what):
            kb.KV8Layer(**{**dict(MAX_BS=1, MAX_LEN=128, H_KV=1, device="cpu"), **bad})


def test_tangents_and_outputs_that_want_a_gradient_are_refused(L):
    """A forward-mode dual would lose its tangent, a lent output that autograd tracks its history."""
    import types

    import torch.autograd.forward_ad as fwd

    import kitty_b200 as kb

    x = torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16)
    rot = types.SimpleNamespace(device=torch.device("cpu"))
    layer = types.SimpleNamespace(device=torch.device("cpu"))
    n = torch.zeros(1, dtype=torch.int32)

    def calls(a, b):
        return [lambda: kb.apply_rotary(a, b, torch.arange(2), rot), lambda: kb.apply_rotary(b, a, torch.arange(2), rot),
                lambda: kb.prompt_attention(a, b, b, 1.0), lambda: kb.prompt_attention(b, a, b, 1.0), lambda: kb.prompt_attention(b, b, a, 1.0),
                lambda: kb.kv8_append(layer, a, b, n), lambda: kb.kv8_append(layer, b, a, n), lambda: kb.kv8_append(layer, b, b, n, query=a),
                lambda: kb.kv8_attention(a[:, :, :1], layer, n, 1.0)]

    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for grad in (torch.enable_grad, torch.no_grad):
            with grad():
                for call in calls(dual, x):
                    with pytest.raises(ValueError, match="no forward derivative"):
                        call()
        L.refuse_gradients("it", x, None)
    want = x.clone().requires_grad_()
    for call in (lambda: kb.apply_rotary(x, x, torch.arange(2), rot, query_out=want), lambda: kb.apply_rotary(x, x, torch.arange(2), rot, key_out=want),
                 lambda: kb.prompt_attention(x, x, x, 1.0, out=want), lambda: kb.kv8_attention(x[:, :, :1], layer, n, 1.0, out=want[:, :, :1])):
        with pytest.raises(ValueError, match="no backward pass"):
            call()


def test_workspaces_are_planned_on_the_tensors_own_device(L, monkeypatch):
    """How a call is split depends on the device's multiprocessors: the library is asked with that device current."""
    import types

    import kitty_b200 as kb
    from kitty_b200 import prompt

    current = ["cuda:0"]

    class Device:
        def __init__(self, dev):
            self.dev = str(dev)

        def __enter__(self):
            current.append(self.dev)

        def __exit__(self, *exc):
            current.pop()

    asked = []
    fake = types.SimpleNamespace(kitty_kv8_workspace_bytes=lambda *a: asked.append((current[-1], a)) or 64,
                                 kitty_prompt_workspace_bytes=lambda *a: asked.append((current[-1], a)) or 64)
    monkeypatch.setattr(L, "lib", lambda: fake)
    monkeypatch.setattr(torch.cuda, "device", Device)
    layer = types.SimpleNamespace(_workspace_need={}, H_KV=2, MAX_PAGE=64, device=torch.device("cuda", 1))
    assert kb.KV8Layer.workspace_bytes(layer, 3, 8) == kb.KV8Layer.workspace_bytes(layer, 3, 8) == 64
    assert prompt._workspace_need(torch.device("cuda", 2), 1, 7, 9, 4, 2, True, False) == 64
    assert asked == [("cuda:1", (3, 2, 8, 64)), ("cuda:2", (1, 7, 9, 4, 2, 1, 0))]
    prompt._workspace_need.cache_clear()
