"""Cases of the prompt-side operators and of the 8-bit cache: inputs, plain forms and exact values.

Operators, with head_dim 128 throughout (the package's geometry):

rotary            apply_rotary: query and key heads turned by position-dependent angles.
prompt_attention  causal attention of a prompt, grouped heads, dense or packed sequences.
kv8_append        one token, a piece or a whole prompt into the paged 8-bit cache, keys rotated on the way;
                  kv8_expand gives the stored tokens back as 16-bit values.
kv8_attention     one query token per sequence against the 8-bit cache.

`run` computes the plain forms with elementary torch operations, or, with `own` true, makes the package's calls.
"""
import math

import torch

own = False

D = 128
BLOCK = 32          # tokens that share a scale in the 8-bit cache
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
# angle scalings for long contexts, in the fields of a model configuration's rope parameters
SCALINGS = {
    "none": None,
    "linear": {"rope_type": "linear", "factor": 4.0},
    "llama3": {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
               "original_max_position_embeddings": 8192},
    "yarn": {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768},
}


# ---- cases ------------------------------------------------------------------------------------------------------ #
def listed():
    return [
        # one token of sixteen sequences deep in a long context: a decode step's rotation, bound by latency
        dict(name="rotary_token", op="rotary", type="bf16", batch=16, tokens=1, hq=32, hkv=8, first=30011, base=500000.0,
             rotary_dim=128, layout="half", scaling="llama3"),
        # prompts of four sequences, as a prefill rotates them before attention: bound by memory
        dict(name="rotary_prompt", op="rotary", type="bf16", batch=4, tokens=4096, hq=32, hkv=8, first=0, base=500000.0,
             rotary_dim=128, layout="half", scaling="none"),
        # a handful of short requests packed together, lengths around a tile's edge: bound by latency
        dict(name="prompt_packed_short", op="prompt", type="f16", hq=28, hkv=4, lengths="1,37,128,129,300", prefix=0,
             packed=True),
        # four full prompts of equal length, the ordinary prefill
        dict(name="prompt_4x4096", op="prompt", type="bf16", hq=32, hkv=8, lengths="4096,4096,4096,4096", prefix=0,
             packed=False),
        # the last piece of a 32768-token prompt that arrives in pieces: every query sees the earlier tokens too
        dict(name="prompt_piece_32k", op="prompt", type="bf16", hq=32, hkv=8, lengths="4096", prefix=28672, packed=False),
        # requests of very different lengths in one packed batch, odd sizes
        dict(name="prompt_packed_ragged", op="prompt", type="f16", hq=28, hkv=4,
             lengths="911,4096,63,2500,1,7007,350,1729", prefix=0, packed=True),
        # a decode step of a full batch: one token per sequence appended, query rotated in the same call
        dict(name="append_token", op="append", type="bf16", batch=128, tokens=1, hq=32, hkv=8, start=32767, spread=9001,
             short=0, base=500000.0, rotary_dim=128, layout="half", scaling="none"),
        # whole prompts quantized into an empty cache: bound by memory
        dict(name="append_prompt", op="append", type="bf16", batch=4, tokens=4096, hq=0, hkv=8, start=0, spread=0, short=0,
             base=500000.0, rotary_dim=128, layout="half", scaling="none"),
        # a ragged piece of a few sequences, half of the head rotated in neighbouring pairs, scaled angles
        dict(name="append_piece_ragged", op="append", type="f16", batch=7, tokens=777, hq=0, hkv=4, start=4096, spread=4096,
             short=500, base=10000.0, rotary_dim=64, layout="interleaved", scaling="yarn"),
        # a single short conversation: bound by latency
        dict(name="attention_short", op="attention", type="bf16", batch=1, hq=32, hkv=8, ctx=517, spread=0),
        # a batch of long contexts: bound by memory
        dict(name="attention_32k", op="attention", type="bf16", batch=32, hq=32, hkv=8, ctx=32768, spread=0),
        # few very long contexts of different lengths, groups of seven heads
        dict(name="attention_131k_g7", op="attention", type="f16", batch=8, hq=28, hkv=4, ctx=131071, spread=65000),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _heads(rng):
    return rng.choice([(32, 8), (28, 4), (16, 16), (8, 1), (40, 8), (32, 2)])


def _angles(rng):
    r = rng.choice([128, 128, 64, 96, 32, 20])
    return dict(base=rng.choice([10000.0, 500000.0, 1000000.0]), rotary_dim=r,
                layout=rng.choice(["half", "half", "interleaved"]), scaling=rng.choice(sorted(SCALINGS)))


def draw(rng):
    op = rng.choice(["rotary", "prompt", "prompt", "append", "attention", "attention"])
    kind = rng.choice(sorted(TYPES))
    hq, hkv = _heads(rng)
    if op == "rotary":
        tokens = _log_int(rng, 1, 4096)
        batch = _log_int(rng, 1, max(1, min(128, 12000 // tokens)))
        return dict(op=op, type=kind, batch=batch, tokens=tokens, hq=hq, hkv=hkv, first=_log_int(rng, 1, 120000) - 1,
                    **_angles(rng))
    if op == "prompt":
        if rng.random() < 0.5:
            n = _log_int(rng, 1, 24)
            lens = [_log_int(rng, 1, 6000) for _ in range(n)]
            while sum(x * x for x in lens) > 48_000_000:
                lens.pop()
            lens = lens or [517]
            return dict(op=op, type=kind, hq=hq, hkv=hkv, lengths=",".join(map(str, lens)), prefix=0, packed=True)
        length = _log_int(rng, 1, 4096)
        prefix = rng.choice([0, 0, 1, _log_int(rng, 1, 12000)])
        batch = _log_int(rng, 1, max(1, min(32, int(4.0e7 // (length * (prefix + length // 2 + 1))), 16000 // (length + prefix))))
        return dict(op=op, type=kind, hq=hq, hkv=hkv, lengths=",".join([str(length)] * batch), prefix=prefix, packed=False)
    if op == "append":
        if rng.random() < 0.4:
            return dict(op=op, type=kind, batch=_log_int(rng, 1, 128), tokens=1, hq=hq, hkv=hkv,
                        start=_log_int(rng, 1, 16000), spread=rng.choice([0, 777]), short=0, **_angles(rng))
        tokens = _log_int(rng, 2, 4096)
        batch = _log_int(rng, 1, max(1, min(32, 12000 // tokens)))
        start = BLOCK * _log_int(rng, 1, 200)
        return dict(op=op, type=kind, batch=batch, tokens=tokens, hq=rng.choice([0, hq]), hkv=hkv, start=start,
                    spread=rng.choice([0, start]), short=rng.choice([0, tokens // 2, tokens]), **_angles(rng))
    ctx = _log_int(rng, 1, 100000)
    batch = _log_int(rng, 1, max(1, min(160, 4_000_000 // (ctx * hkv))))
    return dict(op=op, type=kind, batch=batch, hq=hq, hkv=hkv, ctx=ctx, spread=rng.choice([0, ctx // 3, ctx]))


def _row(case, top, spread, b):
    """Row b's share of a batch whose values fall evenly from `top` to `top - spread`."""
    return top - spread * b // max(case["batch"] - 1, 1)


def _starts(case):
    s = [max(0, _row(case, case["start"], case["spread"], b)) for b in range(case["batch"])]
    return s if case["tokens"] == 1 else [x // BLOCK * BLOCK for x in s]


def _counts(case):
    return [_row(case, case["tokens"], case["short"], b) for b in range(case["batch"])]


def _contexts(case):
    return [_row(case, case["ctx"], case["spread"], b) for b in range(case["batch"])]


def _lengths(case):
    return [int(x) for x in case["lengths"].split(",")]


# ---- inputs ----------------------------------------------------------------------------------------------------- #
def _keys(gen, shape, dtype):
    """Gaussian keys with four channels of each head eight times as large, as trained models have them."""
    k = torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32)
    for h in range(shape[-2]):
        k[..., h, torch.randperm(D, generator=gen, device=DEV)[:4]] *= 8.0
    return k.to(dtype)


def _values(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).to(dtype)


def _queries(gen, shape, dtype):
    return (0.7 * torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32)).to(dtype)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _frequencies(case):
    """(radians per position of each pair in 64 bits, factor on cosine and sine)."""
    r, base, s = case["rotary_dim"], case["base"], SCALINGS[case["scaling"]]
    inv = base ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
    factor = 1.0
    if s is None:
        pass
    elif s["rope_type"] == "linear":
        inv = inv / s["factor"]
    elif s["rope_type"] == "llama3":
        orig, lo, hi = s["original_max_position_embeddings"], s["low_freq_factor"], s["high_freq_factor"]
        turns = orig * inv / (2 * math.pi)
        mix = ((turns - lo) / (hi - lo)).clamp(0.0, 1.0)
        inv = inv / s["factor"] * (1 - mix) + inv * mix
    else:
        orig = s["original_max_position_embeddings"]
        first, last = (r * math.log(orig / (n * 2 * math.pi)) / (2 * math.log(base)) for n in (32.0, 1.0))
        first, last = max(math.floor(first), 0), min(math.ceil(last), r - 1)
        ramp = ((torch.arange(r // 2, dtype=torch.float64) - first) / max(last - first, 0.001)).clamp(0.0, 1.0)
        inv = inv / s["factor"] * ramp + inv * (1 - ramp)
        factor = 0.1 * math.log(s["factor"]) + 1.0
    return inv, factor


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    dtype = TYPES[case["type"]]
    hq, hkv = case["hq"], case["hkv"]
    st = dict(case=case, dtype=dtype)
    if "rotary_dim" in case:
        if own:
            from kitty_b200 import RotaryEmbedding

            st["rotary"] = RotaryEmbedding(D, base=case["base"], rotary_dim=case["rotary_dim"], layout=case["layout"],
                                           scaling=SCALINGS[case["scaling"]], device=DEV)
        inv, st["factor"] = _frequencies(case)
        st["inv"] = inv.to(DEV)
    if case["op"] == "rotary":
        B, T = case["batch"], case["tokens"]
        # the projections' layout [B, T, H, D], handed over as [B, H, T, D] views
        st["q"] = _queries(gen, (B, T, hq, D), dtype).transpose(1, 2)
        st["k"] = _keys(gen, (B, T, hkv, D), dtype).transpose(1, 2)
        st["positions"] = (case["first"] + torch.arange(T, device=DEV))[None, :].repeat(B, 1)
    elif case["op"] == "prompt":
        lens = _lengths(case)
        if case["packed"]:
            total = sum(lens)
            st["q"] = _queries(gen, (total, hq, D), dtype)
            st["k"] = _keys(gen, (total, hkv, D), dtype)
            st["v"] = _values(gen, (total, hkv, D), dtype)
            st["cu"] = _i32([0] + [sum(lens[:i + 1]) for i in range(len(lens))])
        else:
            B, L = len(lens), lens[0]
            st["q"] = _queries(gen, (B, L, hq, D), dtype).transpose(1, 2)
            st["k"] = _keys(gen, (B, L + case["prefix"], hkv, D), dtype).transpose(1, 2)
            st["v"] = _values(gen, (B, L + case["prefix"], hkv, D), dtype).transpose(1, 2)
    elif case["op"] == "append":
        B, T = case["batch"], case["tokens"]
        starts, counts = _starts(case), _counts(case)
        st["k"] = _keys(gen, (B, T, hkv, D), dtype).transpose(1, 2)
        st["v"] = _values(gen, (B, T, hkv, D), dtype).transpose(1, 2)
        st["q"] = _queries(gen, (B, T, hq, D), dtype).transpose(1, 2) if hq else None
        st["start"], st["count"] = _i32(starts), _i32(counts)
        st["after"] = st["start"] + st["count"]
        # the up to 31 tokens of each row's open block, which a single appended token may complete
        st["open_k"] = _keys(gen, (B, BLOCK, hkv, D), dtype).transpose(1, 2).contiguous()
        st["open_v"] = _values(gen, (B, BLOCK, hkv, D), dtype).transpose(1, 2).contiguous()
        if own:
            from kitty_b200 import KV8Layer, kv8_append

            layer = KV8Layer(B, max(starts) + T, hkv, D, dtype=dtype, device=DEV)
            aligned = st["start"] // BLOCK * BLOCK
            kv8_append(layer, st["open_k"], st["open_v"], aligned, lengths=st["start"] - aligned)
            st["layer"] = layer
    else:
        B, ctx = case["batch"], _contexts(case)
        st["q"] = _queries(gen, (B, hq, 1, D), dtype)
        st["lengths"] = _i32(ctx)
        st["scaling"] = D ** -0.5
        if own:
            from kitty_b200 import KV8Layer, kv8_append

            # pages in scattered order, as a cache that has served other requests holds them
            order = torch.randperm(B * -(-max(ctx) // 128), generator=torch.Generator().manual_seed(seed))
            layer = KV8Layer(B, max(ctx), hkv, D, dtype=dtype, device=DEV,
                             page_table=order.view(B, -1).to(device=DEV, dtype=torch.int64))
            st["layer"] = layer
        else:
            st["rows"] = []
        for b, n in enumerate(ctx):
            k = _keys(gen, (max(ctx), hkv, D), dtype)[:n].transpose(0, 1)
            v = _values(gen, (max(ctx), hkv, D), dtype)[:n].transpose(0, 1)
            if own:
                if n:
                    some = torch.zeros(B, dtype=torch.int32, device=DEV)
                    some[b] = n
                    kv8_append(layer, k.unsqueeze(0).expand(B, -1, -1, -1), v.unsqueeze(0).expand(B, -1, -1, -1),
                               torch.zeros_like(some), lengths=some)
            else:
                full = n // BLOCK * BLOCK
                st["rows"].append(_codes(k[:, :full]) + _codes(v[:, :full]) + (k[:, full:].contiguous(), v[:, full:].contiguous()))
    return st


# ---- plain forms ------------------------------------------------------------------------------------------------ #
def _codes(x):
    """Blocks of 32 tokens of [H, n, D] (n a multiple of 32) as whole numbers -127..127 and one scale per block."""
    h, n, _ = x.shape
    x = x.double().reshape(h, n // BLOCK, BLOCK, D)
    top = x.abs().amax(dim=(2, 3))
    t = x * 127.0 / torch.where(top > 0, top, 1.0)[..., None, None]
    codes = torch.sign(t) * torch.floor(t.abs() + 0.5)          # halves away from zero
    scale = torch.where(top > 0, top.float() / 127.0, 1.0)
    return codes.to(torch.int8), scale


def _turn(x, positions, inv, factor, rotary_dim, layout):
    """x [B, H, T, D] turned by positions [B, T]; 32 bits, angles in 64."""
    ang = positions.double()[:, None, :, None] * inv
    ang = ang - torch.round(ang / (2 * math.pi)) * (2 * math.pi)
    c, s = (torch.cos(ang) * factor).float(), (torch.sin(ang) * factor).float()
    r = rotary_dim
    x = x.float()
    a, b = (x[..., :r // 2], x[..., r // 2:r]) if layout == "half" else (x[..., 0:r:2], x[..., 1:r:2])
    ra, rb = a * c - b * s, b * c + a * s
    turned = torch.cat((ra, rb), -1) if layout == "half" else torch.stack((ra, rb), -1).flatten(-2)
    return torch.cat((turned, x[..., r:]), -1)


def _run_rotary(st):
    case, dtype = st["case"], st["dtype"]
    if own:
        from kitty_b200 import apply_rotary

        return list(apply_rotary(st["q"], st["k"], st["positions"], st["rotary"]))
    return [_turn(x, st["positions"], st["inv"], st["factor"], case["rotary_dim"], case["layout"]).to(dtype)
            for x in (st["q"], st["k"])]


def _attend(q, k, v, dtype):
    """q [H_Q, n, D], k/v [H, m, D], the last query sees the last key: [n, H_Q, D]."""
    hq, n, _ = q.shape
    h, m, _ = k.shape
    g = hq // h
    out = torch.empty(n, hq, D, dtype=dtype, device=q.device)
    seen = torch.arange(m, device=q.device)[None, :] <= torch.arange(n, device=q.device)[:, None] + (m - n)
    step = max(1, min(h, (1 << 28) // (g * n * m)))             # key heads at once: at most about 1 GB of scores
    for j in range(0, h, step):
        kj, vj = k[j:j + step].float(), v[j:j + step].float()
        e = kj.shape[0]
        qj = q[j * g:(j + e) * g].float().reshape(e, g * n, D)
        s = torch.matmul(qj, kj.transpose(1, 2)).reshape(e, g, n, m) * D ** -0.5
        s = s.masked_fill(~seen, -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o = torch.matmul((p / p.sum(-1, keepdim=True)).reshape(e, g * n, m), vj)
        out[:, j * g:(j + e) * g] = o.reshape(e * g, n, D).transpose(0, 1).to(dtype)
    return out


def _run_prompt(st):
    case, dtype = st["case"], st["dtype"]
    q, k, v = st["q"], st["k"], st["v"]
    if own:
        from kitty_b200 import prompt_attention

        return prompt_attention(q, k, v, D ** -0.5, cu_seqlens=st.get("cu"))
    if case["packed"]:
        at, parts = 0, []
        for n in _lengths(case):
            parts.append(_attend(*(x[at:at + n].transpose(0, 1) for x in (q, k, v)), dtype))
            at += n
        return torch.cat(parts)
    return torch.stack([_attend(q[b], k[b], v[b], dtype) for b in range(q.shape[0])])


def _run_append(st):
    case, dtype = st["case"], st["dtype"]
    k, v, q = st["k"], st["v"], st["q"]
    B, H, T, _ = k.shape
    if own:
        from kitty_b200 import kv8_append, kv8_expand

        rq = kv8_append(st["layer"], k, v, st["start"], lengths=st["count"], rotary=st["rotary"], query=q)
        ko, vo = kv8_expand(st["layer"], st["after"], T, start=st["start"])
        return [ko, vo] + ([rq] if q is not None else [])
    positions = st["start"][:, None] + torch.arange(T, device=DEV)
    turn = lambda x: _turn(x, positions, st["inv"], st["factor"], case["rotary_dim"], case["layout"]).to(dtype)  # noqa: E731
    out = []
    starts, counts = _starts(case), _counts(case)
    for x, opened in ((turn(k), st["open_k"]), (v, st["open_v"])):
        res = torch.zeros(B, H, T, D, dtype=dtype, device=DEV)
        for b in range(B):
            lead, n = starts[b] % BLOCK, counts[b]
            seq = torch.cat((opened[b, :, :lead], x[b, :, :n]), 1) if lead else x[b, :, :n]
            full = (lead + n) // BLOCK * BLOCK
            if full:
                codes, scale = _codes(seq[:, :full])
                held = (codes.float() * scale[..., None, None]).reshape(H, full, D).to(dtype)
                seq = torch.cat((held, seq[:, full:]), 1)
            res[b, :, :n] = seq[:, lead:]
        out.append(res)
    return out + ([turn(q)] if q is not None else [])


def _run_attention(st):
    case, dtype = st["case"], st["dtype"]
    q = st["q"]
    if own:
        from kitty_b200 import kv8_attention

        return kv8_attention(q, st["layer"], st["lengths"], st["scaling"])
    B, hq, _, _ = q.shape
    h = case["hkv"]
    out = torch.zeros(B, 1, hq, D, dtype=dtype, device=DEV)
    for b, (kc, ks, vc, vs, kt, vt) in enumerate(st["rows"]):
        k = torch.cat(((kc.float() * ks[..., None, None]).reshape(h, -1, D), kt.float()), 1)
        v = torch.cat(((vc.float() * vs[..., None, None]).reshape(h, -1, D), vt.float()), 1)
        if k.shape[1] == 0:
            continue                                             # nothing to see: zeros
        s = torch.matmul(q[b].reshape(h, hq // h, D).float(), k.transpose(1, 2)) * st["scaling"]
        p = torch.exp(s - s.amax(-1, keepdim=True))
        out[b, 0] = torch.matmul(p / p.sum(-1, keepdim=True), v).reshape(hq, D).to(dtype)
    return out


def run(state):
    return {"rotary": _run_rotary, "prompt": _run_prompt, "append": _run_append,
            "attention": _run_attention}[state["case"]["op"]](state)


# ---- the least work --------------------------------------------------------------------------------------------- #
def work(case):
    hq, hkv = case["hq"], case["hkv"]
    if case["op"] == "rotary":
        n = case["batch"] * case["tokens"]
        return {"bytes": n * (hq + hkv) * D * 2 * 2 + 8 * n, "flops": n * (hq + hkv) * case["rotary_dim"] * 3}
    if case["op"] == "prompt":
        lens = _lengths(case)
        rows = sum(lens)
        pairs = sum(n * case["prefix"] + n * (n + 1) // 2 for n in lens)
        keys = rows + case["prefix"] * len(lens)
        return {"bytes": 2 * D * (2 * rows * hq + 2 * keys * hkv), "flops": 4 * D * hq * pairs}
    if case["op"] == "append":
        total = flops = 0
        for s, n in zip(_starts(case), _counts(case)):
            lead = s % BLOCK
            full = (lead + n) // BLOCK * BLOCK
            opened = lead if full else 0                        # tokens of the open block that are read again
            read = (n + opened) * hkv * 2 * D * 2
            written = hkv * 2 * (full * D + full // BLOCK * 4 + (lead + n - full - (lead if not full else 0)) * D * 2)
            expanded = n * hkv * 2 * D * (1 + 2)                # 8-bit values in, 16-bit values out
            total += read + written + expanded + n * hq * D * 4
            flops += n * (hkv + hq) * case["rotary_dim"] * 3 + (full + n) * hkv * 2 * D * 2
        return {"bytes": total, "flops": flops}
    ctx = _contexts(case)
    full = sum(n // BLOCK for n in ctx)
    tail = sum(n % BLOCK for n in ctx)
    return {"bytes": hkv * 2 * (full * (BLOCK * D + 4) + tail * D * 2) + 2 * case["batch"] * hq * D * 2,
            "flops": 4 * D * hq * sum(ctx)}


# ---- exact values ----------------------------------------------------------------------------------------------- #
def _exact_frequencies(case):
    r, base, s = case["rotary_dim"], case["base"], SCALINGS[case["scaling"]]
    inv, factor = [], 1.0
    if s is not None and s["rope_type"] == "yarn":
        factor = 0.1 * math.log(s["factor"]) + 1.0
    for i in range(r // 2):
        w = math.exp(-2.0 * i / r * math.log(base))
        if s is None:
            pass
        elif s["rope_type"] == "linear":
            w /= s["factor"]
        elif s["rope_type"] == "llama3":
            length, orig = 2 * math.pi / w, s["original_max_position_embeddings"]
            if length > orig / s["low_freq_factor"]:
                w /= s["factor"]
            elif length >= orig / s["high_freq_factor"]:
                t = (orig / length - s["low_freq_factor"]) / (s["high_freq_factor"] - s["low_freq_factor"])
                w = (1 - t) * w / s["factor"] + t * w
        else:
            def dim(turns):
                return r * math.log(s["original_max_position_embeddings"] / (turns * 2 * math.pi)) / (2 * math.log(base))
            a, b = max(math.floor(dim(32)), 0), min(math.ceil(dim(1)), r - 1)
            t = min(max((i - a) / max(b - a, 0.001), 0.0), 1.0)
            w = w / s["factor"] * t + w * (1 - t)
        inv.append(w)
    return torch.tensor(inv, dtype=torch.float64, device=DEV), factor


def _exact_turn(case, x, positions):
    w, factor = _exact_frequencies(case)
    z = torch.polar(torch.full_like(w, factor).expand(*positions.shape, -1).contiguous(), positions.double()[..., None] * w)
    y = x.double().clone()
    r = case["rotary_dim"]
    if case["layout"] == "half":
        pair = torch.complex(y[..., :r // 2], y[..., r // 2:r]) * z[:, None]
        y[..., :r // 2], y[..., r // 2:r] = pair.real, pair.imag
    else:
        pair = torch.complex(y[..., 0:r:2], y[..., 1:r:2]) * z[:, None]
        y[..., 0:r:2], y[..., 1:r:2] = pair.real, pair.imag
    return y


def _exact_hold(x):
    """[H, n, D] 16-bit values of whole blocks as the cache holds them."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for i in range(0, x.shape[1], BLOCK):
        blk = x[:, i:i + BLOCK].double()
        top = blk.abs().flatten(1).max(1).values[:, None, None]
        t = torch.where(top > 0, 127.0 * blk / top, torch.zeros_like(blk))
        code = torch.where(t >= 0, torch.floor(t + 0.5), torch.ceil(t - 0.5))
        out[:, i:i + BLOCK] = code * (top / 127.0)
    return out


def _exact_softmax(q, k, v, scaling, offset):
    """q [n, D], k/v [m, D] in 64 bits; row i sees keys 0 .. i + offset."""
    s = (q @ k.T) * scaling
    if offset < k.shape[0] - 1:
        i, j = torch.arange(q.shape[0], device=q.device), torch.arange(k.shape[0], device=q.device)
        s[j[None, :] > i[:, None] + offset] = -math.inf
    return torch.softmax(s, dim=-1) @ v


def exact(case, seed):
    global own
    if case["op"] == "prompt" and work(case)["flops"] > 4.0e13:
        return None
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "rotary":
        return [_exact_turn(case, x, st["positions"]) for x in (st["q"], st["k"])]
    if case["op"] == "prompt":
        def one(q, k, v):                                        # [n, H, D] each
            g = q.shape[1] // k.shape[1]
            res = torch.empty(q.shape, dtype=torch.float64, device=q.device)
            for h in range(q.shape[1]):
                kh, vh = k[:, h // g].double(), v[:, h // g].double()
                for i in range(0, q.shape[0], 2048):
                    part = q[i:i + 2048, h].double()
                    res[i:i + 2048, h] = _exact_softmax(part, kh, vh, D ** -0.5, i + k.shape[0] - q.shape[0])
            return res
        if case["packed"]:
            lens = _lengths(case)
            return torch.cat([one(*t) for t in zip(*(x.split(lens) for x in (st["q"], st["k"], st["v"])))])
        return torch.stack([one(*(x[b].transpose(0, 1) for x in (st["q"], st["k"], st["v"])))
                            for b in range(len(_lengths(case)))])
    if case["op"] == "append":
        B, H, T, _ = st["k"].shape
        pos = st["start"].long()[:, None] + torch.arange(T, device=DEV)[None, :]
        outs = []
        for x, opened in ((_exact_turn(case, st["k"], pos).to(st["dtype"]), st["open_k"]), (st["v"], st["open_v"])):
            res = torch.zeros(B, H, T, D, dtype=torch.float64, device=DEV)
            for b, (s, n) in enumerate(zip(_starts(case), _counts(case))):
                lead = s % BLOCK
                seq = torch.cat((opened[b][:, :lead], x[b][:, :n]), 1)
                full = seq.shape[1] - seq.shape[1] % BLOCK
                seq = torch.cat((_exact_hold(seq[:, :full]), seq[:, full:].double()), 1)
                res[b, :, :n] = seq[:, lead:lead + n]
            outs.append(res)
        return outs + ([_exact_turn(case, st["q"], pos)] if st["q"] is not None else [])
    q = st["q"].double()
    g = case["hq"] // case["hkv"]
    out = torch.zeros(case["batch"], 1, case["hq"], D, dtype=torch.float64, device=DEV)
    for b, (kc, ks, vc, vs, kt, vt) in enumerate(st["rows"]):
        for h in range(case["hkv"]):
            k = torch.cat(((kc[h].double() * ks[h].double()[:, None, None]).reshape(-1, D), kt[h].double()))
            v = torch.cat(((vc[h].double() * vs[h].double()[:, None, None]).reshape(-1, D), vt[h].double()))
            if k.shape[0]:
                out[b, 0, h * g:(h + 1) * g] = _exact_softmax(q[b, h * g:(h + 1) * g, 0], k, v, st["scaling"], k.shape[0])
    return out
