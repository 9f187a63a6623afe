"""The 4-bit KV cache's statements on the CPU: quantiser against a 64-bit search over the representable values,
writer / reader / attention / page copies of `ops` on CPU tensors."""
import math

import pytest
import torch

from vllm_suffix_hybrid_b200 import ops

MAGS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def nearest(grid, x):
    """Index of the nearest grid value, the even index on a tie."""
    dist = (x[..., None] - grid).abs()
    best = dist.min(-1, keepdim=True).values
    tied = dist == best
    idx = torch.arange(grid.numel())
    return torch.where(tied, idx + (idx % 2) * 1000, 1 << 20).min(-1).values % 1000


def test_quantiser_picks_the_nearest_scale_and_codes():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(200, 64, generator=g) * torch.exp(3 * torch.randn(200, 1, generator=g))
    x = torch.cat((x, x.bfloat16().float()))  # bf16 values have ties
    x[0] = 0
    x[1] *= 1e5
    packed, scales = ops.ref.kv_fp4_quantize(x)
    grid = torch.arange(0x7F, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    b = x.double().view(-1, 4, 16)
    want = (b.abs().amax(-1) / 6).clamp(2.0 ** -9, 448.0)
    s = grid[scales.long()]
    # fp32's amax / 6 may cross a midpoint by a rounding: only there may the scale differ
    exact = nearest(grid, want)
    near_tie = ((want - (grid[exact] + grid[scales.long()]) / 2).abs() <= want * 2.0 ** -22)
    assert ((exact == scales) | near_tie).all()
    codes = torch.stack((packed & 15, packed >> 4), -1).flatten(1).view(-1, 4, 16)
    assert torch.equal((codes & 7).long(), nearest(MAGS, (b.abs() / s[..., None]).clamp(max=6.0)))
    assert torch.equal(codes > 7, torch.signbit(b))
    val = ops.ref.kv_fp4_dequantize(packed, scales, 0.5).double().view(-1, 4, 16)
    assert torch.equal(val, torch.where(codes > 7, -1.0, 1.0) * MAGS[(codes & 7).long()] * s[..., None] * 0.5)


def test_write_read_attend_roundtrip():
    hq, hk, d, T = 4, 2, 64, 70
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(T, (hq + 2 * hk) * d, generator=g)
    keep = qkv.clone()
    pos = torch.arange(T)
    cs = ops.ref.rope_cos_sin(128, d, 10000.0)
    k = torch.zeros(ops.kv_fp4_cache_shape(4, hk, d), dtype=torch.uint8)
    v = torch.zeros_like(k)
    bt = torch.tensor([[3, 1]], dtype=torch.int32)
    slots = bt[0].long()[pos // 64] * 64 + pos % 64
    slots[5] = -1
    q = ops.rope_kv_write_fp4(qkv, pos, cs, k, v, slots, hq, hk, d, d, 0.5, 2.0)
    assert torch.equal(qkv, keep)
    rot = ops.ref.apply_rope(qkv[:, : (hq + hk) * d].view(T, hq + hk, d), pos, cs)
    assert torch.allclose(q.view(T, hq, d), rot[:, :hq])
    kr, vr = ops.kv_fp4_read(k, v, slots, d, 0.5, 2.0)
    assert (kr[5] == 0).all() and (vr[5] == 0).all()
    ok = slots >= 0
    # a code is within half a step of its value: at most 1/6 of the block's largest (the step below 6 is 2), and
    # the scale's own rounding (2^-4) may saturate the largest
    for got, want in ((kr, rot[:, hq:]), (vr, qkv[:, (hq + hk) * d:].view(T, hk, d))):
        amax = want.view(T, hk, -1, 16).abs().amax(-1, keepdim=True)
        off = (got - want).view(T, hk, -1, 16).abs()
        assert (off[ok] <= amax[ok] * (1 / 6 + 2.0 ** -4)).all()
    out = torch.empty(3, hq * d)
    ops.paged_attention_fp4(out, q[-3:], k, v, bt, torch.tensor([T]), torch.tensor([0, 3]), hq, d, d ** -0.5, 3, 0.5, 2.0)
    for i in range(3):
        n = T - 2 + i
        kk, vv = kr[:n].repeat_interleave(2, 1), vr[:n].repeat_interleave(2, 1)
        p = torch.softmax(torch.einsum("hd,nhd->hn", q[T - 3 + i].view(hq, d), kk) * d ** -0.5, -1)
        # slot 5 was never written: its page bytes are zeros, as read back
        assert torch.allclose(out[i].view(hq, d), torch.einsum("hn,nhd->hd", p, vv), atol=1e-5)


def test_rows_without_keys_are_zero():
    k = torch.zeros(ops.kv_fp4_cache_shape(2, 1, 64), dtype=torch.uint8)
    out = torch.full((3, 64), math.nan)
    ops.paged_attention_fp4(out, torch.randn(3, 64), k, k, torch.zeros(2, 1, dtype=torch.int32), torch.tensor([0, 1]),
                            torch.tensor([0, 1, 3]), 1, 64, 0.1, 2)
    assert (out == 0).all()


def test_copy_pages_and_shapes():
    c = [torch.arange(6.0)[:, None].expand(6, 4).clone(), torch.arange(12).view(6, 2)]
    ops.copy_kv_pages(c, torch.tensor([1, 2, -1]), torch.tensor([4, 99, 3]))
    assert c[0][:, 0].tolist() == [0, 1, 2, 3, 1, 5] and c[1][4].tolist() == [2, 3]
    ops.copy_kv_pages([], torch.tensor([1]), torch.tensor([2]))
    assert ops.kv_fp4_cache_shape(10, 8, 128) == (10, 8, 4608)
    with pytest.raises(ValueError):
        ops.kv_fp4_cache_shape(10, 8, 96)
