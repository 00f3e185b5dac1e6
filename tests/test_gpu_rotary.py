"""Rotary positions against the formula in 64 bits."""
import pytest
import torch

from tests.ops_ref import rotate, rotate_bound

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}
LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}


@pytest.fixture(scope="module")
def kb():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import kitty_b200

    return kitty_b200


def _check(got, x, pos, rot, layout):
    want = rotate(x, pos, rot.inv_freq.to(DEV), rot.factor, rot.rotary_dim, layout)
    bound = rotate_bound(x, want, abs(rot.factor), rot.rotary_dim, layout, pos, rot.inv_freq.to(DEV))
    off = (got.double() - want).abs()
    assert (off <= bound).all(), ((off - bound).max().item(), off.max().item())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("r", [128, 64, 96, 20, 2, 36])
def test_rotation(kb, dtype, layout, r):
    g = torch.Generator(device=DEV).manual_seed(r)
    B, T, hq, h = 2, 11, 5, 3
    rot = kb.RotaryEmbedding(128, base=10000.0, rotary_dim=r, layout=layout, scaling=YARN if r == 64 else None, device=DEV)
    q = torch.randn(B, T, hq, 128, generator=g, device=DEV).to(dtype).transpose(1, 2)
    k = torch.randn(B, T, h, 128, generator=g, device=DEV).to(dtype).transpose(1, 2)
    pos = torch.tensor([[0, 1, 2, 1000003, 7, 131071, 2 ** 31 + 5, 3, 3, 99999, 4]], device=DEV).repeat(B, 1)
    pos[1] += 17
    qo, ko = kb.apply_rotary(q, k, pos, rot)
    assert qo.shape == q.shape and qo.stride() == q.stride()
    _check(qo, q, pos, rot, layout)
    _check(ko, k, pos, rot, layout)
    assert torch.equal(qo[..., r:], q[..., r:])                       # what does not turn keeps its bits
    # in place, from a fused projection's slices
    fused = torch.cat((q.transpose(1, 2), k.transpose(1, 2)), dim=2)
    fq, fk = fused[:, :, :hq].transpose(1, 2), fused[:, :, hq:].transpose(1, 2)
    a, b = kb.apply_rotary(fq, fk, pos, rot, query_out=fq, key_out=fk)
    assert a is fq and torch.equal(fq, qo) and torch.equal(fk, ko) and torch.equal(b, ko)


@pytest.mark.parametrize("B,T,hq,h", [(1, 1, 32, 8), (16, 1, 28, 4), (3, 257, 8, 1), (1, 8, 1, 1), (0, 4, 2, 2), (2, 0, 2, 2)])
def test_shapes(kb, B, T, hq, h):
    g = torch.Generator(device=DEV).manual_seed(7)
    rot = kb.RotaryEmbedding(base=500000.0, scaling=LLAMA3, device=DEV)
    q = torch.randn(B, hq, T, 128, generator=g, device=DEV).bfloat16()
    k = torch.randn(B, h, T, 128, generator=g, device=DEV).bfloat16()
    pos = torch.arange(T, device=DEV) + 30000
    qo, ko = kb.apply_rotary(q, k, pos, rot)
    if B and T:
        _check(qo, q, pos[None].expand(B, -1), rot, "half")
        _check(ko, k, pos[None].expand(B, -1), rot, "half")


def test_untouched_channels_may_hold_anything(kb):
    rot = kb.RotaryEmbedding(rotary_dim=64, layout="interleaved", device=DEV)
    q = torch.randn(1, 2, 3, 128, device=DEV).half()
    q[..., 64] = float("inf")
    q[..., 100] = float("nan")
    k = q.clone()
    qo, _ = kb.apply_rotary(q, k, torch.arange(3, device=DEV), rot)
    assert torch.isfinite(qo[..., :64]).all()
    assert torch.equal(qo[..., 64:].view(torch.int16), q[..., 64:].view(torch.int16))


def test_captured_and_on_another_stream(kb):
    rot = kb.RotaryEmbedding(device=DEV)
    q, k = torch.randn(2, 4, 1, 128, device=DEV).half(), torch.randn(2, 2, 1, 128, device=DEV).half()
    pos = torch.tensor([[5], [9]], device=DEV)
    want = kb.apply_rotary(q, k, pos, rot)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = kb.apply_rotary(q, k, pos, rot)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = kb.apply_rotary(q, k, pos, rot)
    pos += 100
    graph.replay()
    later = kb.apply_rotary(q, k, pos, rot)
    assert torch.equal(cap[0], later[0]) and torch.equal(cap[1], later[1])


def test_agrees_with_the_decode_token_path(kb):
    """The same rotation as rope_decode_token, whose products are rounded one by one."""
    from kitty_b200.hf_adapter import rope_decode_token

    rot = kb.RotaryEmbedding(device=DEV)
    q, k = torch.randn(3, 1, 8, 128, device=DEV).bfloat16(), torch.randn(3, 1, 2, 128, device=DEV).bfloat16()
    pos = torch.tensor([[4], [77], [1200]], device=DEV)
    ang = pos.double()[..., None] * rot.inv_freq.to(DEV)
    ang = torch.cat((ang, ang), -1)
    a, b = rope_decode_token(q, k, torch.cos(ang).bfloat16(), torch.sin(ang).bfloat16())
    c, d = kb.apply_rotary(q.transpose(1, 2), k.transpose(1, 2), pos, rot)
    # cos and sin rounded to bf16 (2^-8 each of at most |x|), products and sum half a step each
    for x, y, src in ((a, c, q), (b, d, k)):
        s = src.transpose(1, 2).float().abs()
        bound = 6 * 2.0 ** -8 * (s + torch.roll(s, 64, -1))
        assert ((x.float() - y.float()).abs() <= bound + 1e-6).all()


def test_rows_off_their_boundaries(kb):
    rot = kb.RotaryEmbedding(device=DEV)
    wide = torch.randn(2, 3, 5, 129, device=DEV).half()
    q, k = wide[..., 1:], torch.randn(2, 1, 5, 128, device=DEV).half()
    pos = torch.arange(5, device=DEV)
    a, _ = kb.apply_rotary(q, k, pos, rot)
    b, _ = kb.apply_rotary(q.contiguous(), k, pos, rot)
    assert torch.equal(a, b)
    e, _ = kb.apply_rotary(k.expand(2, 4, 5, 128), k, pos, rot)             # one head read four times
    assert torch.equal(e, kb.apply_rotary(k, k, pos, rot)[0].expand(2, 4, 5, 128))
    before = wide.clone()
    for bad in (q, k.expand(2, 3, 5, 128)):
        with pytest.raises(ValueError):
            kb.apply_rotary(q, k, pos, rot, query_out=bad)
    buf = torch.randn(2, 3, 6, 128, device=DEV).half()
    with pytest.raises(ValueError, match="overlaps"):
        kb.apply_rotary(buf[:, :, :5], k, pos, rot, query_out=buf[:, :, 1:])
    assert torch.equal(wide, before)


def test_outputs_beside_the_inputs_in_one_buffer(kb):
    """Slices of one fused projection, turned in place and into other slices of the same buffer."""
    rot = kb.RotaryEmbedding(device=DEV)
    fused = torch.randn(2, 40, 24, 128, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV).bfloat16()
    cut = lambda x, a, b: x[:, :, a:b].transpose(1, 2)                  # noqa: E731
    pos = torch.arange(40, device=DEV)
    want = kb.apply_rotary(cut(fused, 0, 8), cut(fused, 8, 12), pos, rot)
    got = kb.apply_rotary(cut(fused, 0, 8), cut(fused, 8, 12), pos, rot, query_out=cut(fused, 12, 20), key_out=cut(fused, 20, 24))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    a, b = cut(fused, 0, 8), cut(fused, 8, 16)
    before = fused.clone()
    with pytest.raises(ValueError, match="overlaps"):
        kb.apply_rotary(a, b, pos, rot, query_out=b, key_out=a)
    assert torch.equal(fused, before)
