"""The decode-path QKV consumer into E4M3 caches against its BF16 form (bit-identical to the reference's kernel): Q has the same bits,
V codes are the BF16 values' own, K codes lie within a code's half step and the BF16 form's half step of its values."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _call(atlas, torch, fp8, qkv, w, pos, freq, slots, n_slots, t, hq, hk, d, rot, page, k_inv, v_inv, offset_one):
    stride, buf = qkv.shape[1], qkv.clone()
    shape = (-(-n_slots // page), page, hk, d)
    kc, vc = (torch.full(shape, 0x55, dtype=torch.uint8, device="cuda") if fp8 else torch.full(shape, 9.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    base = buf.data_ptr()
    args = (base, base + 2 * hq * d, base + 2 * (hq + hk) * d, stride, stride, w[0], w[1], pos, freq, slots, kc, vc, t, hq, hk, d, rot, page, 1e-6)
    if fp8:
        atlas.qkv_norm_rope_cache_write_fp8(*args, k_inv, v_inv, attention_factor=1.1, norm_offset_one=offset_one)
    else:
        atlas.qkv_norm_rope_cache_write(*args, attention_factor=1.1, norm_offset_one=offset_one)
    torch.cuda.synchronize()
    return buf, kc.view(-1, hk, d), vc.view(-1, hk, d)


@pytest.mark.parametrize("d,rot,hq,hk", [(128, 128, 8, 2), (128, 64, 32, 8), (64, 64, 4, 4), (256, 64, 16, 2), (256, 256, 2, 1), (96, 32, 3, 1), (128, 0, 4, 1), (64, 48, 5, 5),
                                         (50, 20, 2, 1), (224, 128, 2, 2)])
@pytest.mark.parametrize("tokens", [1, 77])
def test_against_the_bf16_form(cuda, atlas, d, rot, hq, hk, tokens):
    torch = cuda
    rng = np.random.default_rng(d + rot + tokens)
    g = torch.Generator(device="cuda")
    g.manual_seed(d + rot)
    width = (hq + 2 * hk) * d
    qkv = (torch.randn((tokens, width + 6), generator=g, device="cuda") * torch.exp2(torch.rand((tokens, 1), generator=g, device="cuda") * 8 - 4)).to(torch.bfloat16)
    w = [(torch.randn(d, generator=g, device="cuda") * 0.2).to(torch.bfloat16) for _ in range(2)]
    pos = torch.from_numpy(rng.integers(0, 131072, tokens).astype(np.int32)).cuda()
    freq = (1e6 ** (-torch.arange(0, max(rot, 2), 2, dtype=torch.float64, device="cuda") / max(rot, 2))).float()
    n_slots = tokens + 20
    slots_np = rng.permutation(n_slots)[:tokens].astype(np.int64)
    slots_np[rng.random(tokens) < 0.1] = -1
    slots = torch.from_numpy(slots_np).cuda()
    k_inv, v_inv, page = 30.0, 50.0, 8
    args = (qkv, w, pos, freq, slots, n_slots, tokens, hq, hk, d, rot, page, k_inv, v_inv, bool(d % 64))
    buf, kc, vc = _call(atlas, torch, False, *args)
    buf8, kc8, vc8 = _call(atlas, torch, True, *args)
    assert torch.equal(buf.view(torch.int16), buf8.view(torch.int16))                            # Q, and K and V as they were
    live = slots[slots >= 0]
    still = torch.ones(kc8.shape[0], dtype=torch.bool, device="cuda")
    still[live] = False
    assert (kc8[still] == 0x55).all() and (vc8[still] == 0x55).all()
    want_v = (vc[live].float() * v_inv).clamp(-448, 448).to(torch.float8_e4m3fn)
    assert torch.equal(vc8[live], want_v.view(torch.uint8))
    # K: the code is within half a step (2^-4 of the value, or 2^-10 below the smallest normal code) of value * inv_scale, whose BF16
    # form is within 2^-8 of it; the product's own rounding is 2^-24; saturation at 448
    near = kc[live].double() * k_inv
    got = kc8[live].view(torch.float8_e4m3fn).double()
    far = near.abs() * (1 + 2.0 ** -8 + 2.0 ** -20)                                              # what the unrounded product may be
    fine = far < 448
    assert ((got - near).abs() <= far * (2.0 ** -4 + 2.0 ** -8 + 2.0 ** -20) + 2.0 ** -10)[fine].all()
    assert (got.abs()[near.abs() * (1 - 2.0 ** -7) > 448] == 448).all()
    passing = list(range(rot, d))
    if passing:                                                                                  # no rotation: the BF16 value itself
        want = (kc[live][..., passing].float() * k_inv).clamp(-448, 448).to(torch.float8_e4m3fn)
        assert torch.equal(kc8[live][..., passing], want.view(torch.uint8))


def test_nan_and_infinity(cuda, atlas):
    """A NaN is a NaN code; an infinity saturates."""
    torch = cuda
    qkv = torch.ones((2, 3 * 64), dtype=torch.bfloat16, device="cuda")
    qkv[0, 130], qkv[1, 131], qkv[1, 132] = float("nan"), float("inf"), float("-inf")
    w = [torch.zeros(64, dtype=torch.bfloat16, device="cuda")] * 2
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    freq = torch.ones(32, dtype=torch.float32, device="cuda")
    slots = torch.arange(2, device="cuda")
    _, kc, vc = _call(atlas, torch, True, qkv, w, pos, freq, slots, 2, 2, 1, 1, 64, 64, 2, 1.0, 1.0, True)
    v = vc.view(torch.float8_e4m3fn).float().view(2, 64)
    assert torch.isnan(v[0, 2]) and v[1, 3] == 448 and v[1, 4] == -448
    assert torch.isfinite(v).sum() == 127
