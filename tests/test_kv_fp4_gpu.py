"""The 4-bit KV cache on the GPU: writer, reader, paged attention, page copies.

The oracle works in 64 bits on the bytes of the pages.  Attention tolerance, per element: the output's rounding to
bf16 (2^-8 |o|); P's rounding to f16 (unit roundoff 2^-11 on every term of sum p |v|, and 2^-25 in absolute terms for
each key whose p is below f16's normal range); 2^-18 of sum p |v| for exp2's approximation and the fp32 sums; and the
fp32 scores, D/16 + 2 roundings of at most 2^-23 of sum |q k| scale each, which move a p relative to the others by up to
twice that.
"""
import math

import pytest
import torch

from vllm_suffix_hybrid_b200 import ops

pytestmark = pytest.mark.gpu

HEADS = [(32, 8, 128), (4, 4, 64), (4, 2, 64), (16, 2, 256), (7, 1, 128), (8, 8, 128), (12, 2, 128), (40, 1, 64)]


def rows64(pages, d, scale):
    """fp64 [n * 64, D] of one head's pages [n, bytes]."""
    split = 32 * d
    b = pages[:, :split].reshape(-1, d // 2).long()
    codes = torch.stack((b & 15, b >> 4), -1).flatten(1)
    mag = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)[codes & 7]
    s = pages[:, split:].reshape(-1, d // 16).view(torch.float8_e4m3fn).double().repeat_interleave(16, 1)
    return torch.where(codes > 7, -mag, mag) * s * scale


def random_cache(blocks, hk, d, seed, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(blocks, hk, 64, d, generator=g) * gain * torch.exp(0.5 * torch.randn(d, generator=g))
    codes, scales = ops.ref.kv_fp4_quantize(x)
    return torch.cat((codes.flatten(2), scales.flatten(2)), 2).contiguous()


def case(q_lens, seqs, hq, hk, d, seed=0, spare=3, cols=None, gain=1.0):
    """Random pages, a shuffled block table, the bytes past each length set to 0xFF (a NaN scale)."""
    g = torch.Generator().manual_seed(seed + 1000)
    need = [(s + 63) // 64 for s in seqs]
    blocks = sum(need) + spare
    k, v = random_cache(blocks, hk, d, seed, gain), random_cache(blocks, hk, d, seed + 1)
    ids = torch.randperm(blocks, generator=g)
    bt = torch.full((len(seqs), max(max(need), 1) if cols is None else cols), 0, dtype=torch.int32)
    at = 0
    for i, (n, s) in enumerate(zip(need, seqs)):
        bt[i, :n] = ids[at:at + n].int()
        at += n
        if s % 64:
            for c in (k, v):
                codes, scales = ops.ref._kv_fp4_views(c, d)
                codes[bt[i, n - 1], :, s % 64:] = 0xFF
                scales[bt[i, n - 1], :, s % 64:] = 0xFF
    q = (torch.randn(sum(q_lens), hq * d, generator=g) * 2).bfloat16()
    qs = torch.tensor([0] + list(q_lens)).cumsum(0)
    return dict(q=q, k=k, v=v, bt=bt, seqs=torch.tensor(seqs), qs=qs, hq=hq, hk=hk, d=d, scale=1 / math.sqrt(d),
                max_q=max(max(q_lens), 1), gk=0.75, gv=1.5)


def oracle(c):
    """(fp64 output, tolerance) [T, hq, D]."""
    hq, hk, d = c["hq"], c["hk"], c["d"]
    T = c["q"].shape[0]
    out, tol = torch.zeros(T, hq, d, dtype=torch.float64), torch.zeros(T, hq, d, dtype=torch.float64)
    for b in range(c["seqs"].numel()):
        s0, s1, n = int(c["qs"][b]), int(c["qs"][b + 1]), int(c["seqs"][b])
        if s1 == s0 or n == 0:
            continue
        used = c["bt"][b, : (n + 63) // 64].long()
        pos = torch.arange(n - (s1 - s0), n)
        seen = torch.arange(n) <= pos[:, None]
        for h in range(hk):
            k, v = rows64(c["k"][used, h], d, c["gk"])[:n], rows64(c["v"][used, h], d, c["gv"])[:n]
            hs = slice(h * hq // hk, (h + 1) * hq // hk)
            sc = torch.einsum("tgd,nd->tgn", c["q"][s0:s1].view(-1, hq, d)[:, hs].double(), k) * c["scale"]
            p = torch.softmax(torch.where(seen[:, None], sc, -math.inf), -1)
            p = torch.where(seen.any(1)[:, None, None], p, 0.0)
            out[s0:s1, hs] = p @ v
            size = torch.einsum("tgd,nd->tgn", c["q"][s0:s1].view(-1, hq, d)[:, hs].double().abs(), k.abs()) * abs(c["scale"])
            score = 2 * (d / 16 + 2) * 2.0 ** -23 * torch.where(seen[:, None], size, 0.0).amax(-1, keepdim=True)
            tol[s0:s1, hs] = (2.0 ** -11 + 2.0 ** -18 + score) * (p @ v.abs()) + n * 2.0 ** -25 * v.abs().max()
    return out, tol + 2.0 ** -8 * out.abs() + 1e-9


def attend(c, q=None, out=None, **kw):
    dev = {n: c[n].cuda() for n in ("k", "v", "bt", "seqs", "qs")}
    q = c["q"].cuda() if q is None else q
    out = torch.full((q.shape[0], c["hq"] * c["d"]), math.nan, dtype=torch.bfloat16, device="cuda") if out is None else out
    ops.paged_attention_fp4(out, q, dev["k"], dev["v"], dev["bt"], dev["seqs"], dev["qs"], c["hq"], c["d"], c["scale"],
                            kw.get("max_q", c["max_q"]), c["gk"], c["gv"])
    return out


def check(c, got):
    want, tol = oracle(c)
    off = (got.cpu().double().view_as(want) - want).abs() - tol
    assert torch.isfinite(got).all()
    assert (off <= 0).all(), f"{(off > 0).sum()} of {off.numel()} beyond the tolerance, worst by {off.max()}"


# ----------------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("hq,hk,d", HEADS)
@pytest.mark.parametrize("seqs", [(1,), (64,), (65, 1, 63), (1000, 17, 128, 129, 2047)])
def test_decode(hq, hk, d, seqs):
    c = case([1] * len(seqs), seqs, hq, hk, d, seed=d + len(seqs))
    check(c, attend(c))


@pytest.mark.parametrize("hq,hk,d", HEADS)
def test_verify_window_ragged(hq, hk, d):
    q = (6, 1, 3, 6, 2)
    c = case(q, (6, 300, 64, 1029, 66), hq, hk, d, seed=3)
    check(c, attend(c))


@pytest.mark.parametrize("hq,hk,d", [(32, 8, 128), (4, 2, 64), (16, 2, 256), (7, 1, 128)])
@pytest.mark.parametrize("q,seqs", [((200,), (200,)), ((65, 130, 1), (65, 400, 90)), ((33, 257), (1000, 257))])
def test_prefill_and_chunks(hq, hk, d, q, seqs):
    c = case(q, seqs, hq, hk, d, seed=5)
    check(c, attend(c))


@pytest.mark.parametrize("hq,hk,d", [(32, 8, 128), (4, 4, 64), (7, 1, 128), (40, 1, 64), (12, 2, 128)])
@pytest.mark.parametrize("q,seqs", [((33,), (33,)), ((64, 17), (9000, 129)), ((129, 257, 1, 0, 63), (129, 300, 5000, 40, 64)),
                                    ((700,), (1500,))])
def test_many_rows(hq, hk, d, q, seqs):
    """Row tiles of one to many rows, one or both halves of a unit, units split over several CTAs and many in one."""
    c = case(q, seqs, hq, hk, d, seed=20 + d)
    check(c, attend(c))


@pytest.mark.parametrize("hq,hk,d", [(32, 8, 128), (4, 4, 64), (16, 2, 256), (7, 1, 128), (40, 1, 64)])
@pytest.mark.parametrize("q,seqs", [((90,), (100,)), ((90,), (256,)), ((70,), (320,)), ((70, 66, 1, 0), (30, 513, 255, 70)),
                                    ((130,), (2048,)), ((3, 40, 0, 129), (300, 0, 900, 129))])
def test_many_rows_in_a_wide_table(hq, hk, d, q, seqs):
    """A table far wider than its lengths says that the work may be large: few short units for many CTAs."""
    c = case(q, seqs, hq, hk, d, seed=30 + d, cols=4000)
    check(c, attend(c))


def test_many_rows_that_see_nothing():
    c = case((90, 70, 40), (30, 0, 40), 8, 2, 128, seed=21)
    got = attend(c)
    check(c, got)
    assert (got[:60] == 0).all() and (got[90:160] == 0).all() and (got[60:90] != 0).any(1).all()


@pytest.mark.parametrize("d", [64, 128, 256])
def test_many_rows_with_a_rising_maximum(d):
    """Keys that grow along the sequence: the softmax reference moves in almost every tile, inside tiles too."""
    c = case((150,), (1500,), 4, 2, d, seed=22)
    x = torch.randn(c["k"].shape[0], 2, 64, d, generator=torch.Generator().manual_seed(22))
    n = c["bt"].shape[1]
    x[c["bt"][0].long()] *= (torch.arange(n * 64).view(n, 1, 64, 1) / 100.0).exp2().clamp(max=400.0)
    codes, scales = ops.ref.kv_fp4_quantize(x)
    c["k"] = torch.cat((codes.flatten(2), scales.flatten(2)), 2).contiguous()
    c["q"] *= torch.logspace(-20, 3, 150, base=2.0)[:, None].bfloat16()
    check(c, attend(c))


@pytest.mark.parametrize("scale", [0.0, -0.125])
@pytest.mark.parametrize("q", [1, 100])
def test_zero_and_negative_scale(scale, q):
    c = case((q,), (300,), 8, 2, 128, seed=23)
    c["scale"] = scale
    check(c, attend(c))


def test_long_context_split_over_many_ctas():
    c = case((1, 2), (40001, 20000), 8, 2, 128, seed=6)
    check(c, attend(c))


def test_rows_that_see_nothing_are_zero():
    """No keys at all, no queries, and more queries than keys (the first rows precede the sequence)."""
    c = case((1, 0, 5, 2), (0, 70, 3, 64), 8, 2, 128, seed=7)
    got = attend(c)
    check(c, got)
    assert (got[0] == 0).all() and (got[1:3] == 0).all() and (got[3:] != 0).any(1).all()


def test_one_dominant_key_and_large_scores():
    """Scores of several thousand: the softmax reference must follow them up, and queries of very different sizes
    must keep their precision."""
    c = case((1, 6), (500, 700), 8, 2, 128, seed=8, gain=20.0)
    c["q"] *= torch.logspace(-30, 2, 7, base=2.0)[:, None].bfloat16()
    check(c, attend(c))


def test_strided_rows_and_tables():
    c = case((3, 1), (300, 41), 8, 2, 128, seed=9)
    hq, d, T = 8, 128, 4
    wide = torch.randn(T, 2 * hq * d + 64, device="cuda").bfloat16()
    wide[:, 64:64 + hq * d] = c["q"].cuda()
    outw = torch.zeros(T, hq * d + 8, dtype=torch.bfloat16, device="cuda")
    bt = torch.zeros(2, c["bt"].shape[1] + 5, dtype=torch.int32)
    bt[:, : c["bt"].shape[1]] = c["bt"]
    full = bt.cuda()[:, : c["bt"].shape[1]]
    got = outw[:, : hq * d]
    ops.paged_attention_fp4(got, wide[:, 64:64 + hq * d], c["k"].cuda(), c["v"].cuda(), full, c["seqs"].cuda(),
                            c["qs"].cuda(), hq, d, c["scale"], 3, c["gk"], c["gv"])
    check(c, got)
    assert (outw[:, hq * d:] == 0).all()


def test_a_short_max_q_len_changes_speed_only():
    c = case((9, 30), (300, 41), 8, 2, 128, seed=10)
    check(c, attend(c, max_q=1))


def test_bad_block_ids_stay_in_bounds():
    """Ids outside the cache read block 0 (whatever it holds); only the rows that use them are affected."""
    c = case((1, 1), (300, 200), 8, 2, 128, seed=11)
    c["bt"][0, 1] = 1 << 30
    c["bt"][0, 2] = -7
    got = attend(c)
    c["bt"][0, 1:3] = 0
    same = attend(c)
    assert torch.equal(got.view(torch.int16), same.view(torch.int16))  # bits: block 0 holds NaN scales in this case
    check(dict(c, q=c["q"][1:], bt=c["bt"][1:], seqs=c["seqs"][1:], qs=torch.tensor([0, 1])), got[1:])


def test_repeats_are_identical_and_streams_do_not_disturb_each_other():
    a, b = case((1,) * 9, (3000,) * 9, 8, 2, 128, seed=12), case((2,) * 5, (5000,) * 5, 16, 2, 256, seed=13)
    ra, rb = attend(a), attend(b)
    check(a, ra)
    check(b, rb)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(attend((a, b)[i % 2]))
    torch.cuda.synchronize()
    for i, r in enumerate(got):
        assert torch.equal(r, (ra, rb)[i % 2])


def test_graph_replay_follows_lengths():
    """A captured call reads lengths and tables at replay, as the engine's decode graphs do."""
    c = case((1, 1, 1), (3000, 2000, 1500), 32, 8, 128, seed=14)
    dev = {n: c[n].cuda() for n in ("k", "v", "bt", "seqs", "qs", "q")}
    out = torch.empty(3, 32 * 128, dtype=torch.bfloat16, device="cuda")

    def call():
        for _ in range(2):  # two layers of a step share the capture's scratch
            ops.paged_attention_fp4(out, dev["q"], dev["k"], dev["v"], dev["bt"], dev["seqs"], dev["qs"], 32, 128,
                                    c["scale"], 1, c["gk"], c["gv"])

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for seqs in ((3000, 2000, 1500), (1, 2000, 64), (2990, 5, 700)):
        c["seqs"] = torch.tensor(seqs)
        dev["seqs"].copy_(c["seqs"])
        for _ in range(2):
            out.fill_(math.nan)
            graph.replay()
        torch.cuda.synchronize()
        # bytes past a length are another token's here, not 0xFF: the oracle reads only the length's own
        check(c, out)


def test_batch_invariant_mode(monkeypatch):
    """A row's bits do not depend on the window's width or on the other requests."""
    monkeypatch.setenv("SH_BATCH_INVARIANT", "1")
    c = case((5, 1, 3), (900, 700, 64), 8, 2, 128, seed=15)
    all_rows = attend(c)
    check(c, all_rows)
    for t in range(5):  # request 0's window, one token at a time
        one = dict(c, q=c["q"][t:t + 1], seqs=torch.tensor([900 - 4 + t]), bt=c["bt"][:1], qs=torch.tensor([0, 1]))
        assert torch.equal(attend(one, max_q=1)[0], all_rows[t])


def test_refusals():
    c = case((1,), (100,), 8, 2, 128, seed=16)
    q, k, v, bt = c["q"].cuda(), c["k"].cuda(), c["v"].cuda(), c["bt"].cuda()
    sl, qs = c["seqs"].cuda(), c["qs"].cuda()

    def call(**kw):
        a = dict(out=torch.empty_like(q), q=q, k=k, v=v, bt=bt, sl=sl, qs=qs, hq=8, d=128, mq=1, gk=1.0)
        a.update(kw)
        ops.paged_attention_fp4(a["out"], a["q"], a["k"], a["v"], a["bt"], a["sl"], a["qs"], a["hq"], a["d"], 0.1, a["mq"],
                                a["gk"], 1.0)

    call()
    buf = torch.zeros(2, 8 * 128 + 4, dtype=torch.bfloat16, device="cuda")
    for kw in (dict(q=q.half()), dict(q=q.float()), dict(hq=7), dict(d=64), dict(d=96), dict(k=k[:, :, :-16]),
               dict(k=k.view(torch.int8)), dict(bt=bt.long()), dict(sl=sl.int()), dict(qs=qs[:1]), dict(mq=0),
               dict(gk=0.0), dict(out=torch.empty_like(q, dtype=torch.float32)), dict(q=buf[:1, 4:]),
               dict(v=v[:1]), dict(bt=c["bt"]), dict(k=k[..., ::2])):
        with pytest.raises((RuntimeError, TypeError)):
            call(**kw)


# ----------------------------------------------------------------------------------------------- writer and reader
def write_case(T, hq, hk, d, rot, seed=0, pad=0, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(T, (hq + 2 * hk) * d + pad, generator=g) * gain).bfloat16()
    pos = torch.randint(0, 512, (T,), generator=g)
    ang = torch.arange(512)[:, None].double() / 1000.0 ** (torch.arange(0, rot, 2).double() / max(rot, 1))
    cs = torch.cat((ang.cos(), ang.sin()), 1).float()
    blocks = T // 64 + 3
    slots = torch.randperm(blocks * 64, generator=g)[:T]
    shape = ops.kv_fp4_cache_shape(blocks, hk, d)
    return qkv, pos, cs, slots, torch.full(shape, 0xAB, dtype=torch.uint8), torch.full(shape, 0xCD, dtype=torch.uint8)


@pytest.mark.parametrize("hq,hk,d,rot", [(32, 8, 128, 128), (16, 2, 256, 64), (4, 2, 64, 64), (7, 1, 128, 24), (8, 8, 64, 0),
                                         (4, 1, 256, 256), (2, 2, 128, 96)])
@pytest.mark.parametrize("T", [1, 37])
def test_write_matches_the_reference_bit_for_bit(hq, hk, d, rot, T):
    """Every operation up to the codes is rounded alike on both sides, so queries, codes and scales are equal, and so
    is every byte that no slot names."""
    qkv, pos, cs, slots, k, v = write_case(T, hq, hk, d, rot, seed=T, pad=8 * (T % 2))
    if T > 5:
        slots[3], slots[5] = -1, 1 << 40
    kd, vd = k.cuda(), v.cuda()
    src = qkv.cuda()
    q = ops.rope_kv_write_fp4(src, pos.cuda(), cs.cuda(), kd, vd, slots.cuda(), hq, hk, d, rot, 0.75, 2.0)
    want = ops.rope_kv_write_fp4(qkv, pos, cs, k, v, slots, hq, hk, d, rot, 0.75, 2.0)
    assert torch.equal(src.cpu(), qkv)
    assert torch.equal(q.cpu(), want)
    assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v)
    kr, vr = ops.kv_fp4_read(kd, vd, slots.cuda(), d, 0.75, 2.0)
    kw, vw = ops.kv_fp4_read(k, v, slots, d, 0.75, 2.0)
    assert torch.equal(kr.cpu(), kw.bfloat16()) and torch.equal(vr.cpu(), vw.bfloat16())


def test_write_extremes():
    """Zeros, the smallest and largest magnitudes, infinities and NaN: the cache stays finite."""
    hq, hk, d = 2, 2, 128
    qkv, pos, cs, slots, k, v = write_case(8, hq, hk, d, 0, seed=4)
    qkv[0] = 0
    qkv[1] = -0.0
    qkv[2] = 1e-30
    qkv[3] = 3e38
    qkv[4, ::3] = math.inf
    qkv[5, ::5] = -math.inf
    qkv[6, ::7] = math.nan
    qkv[7] = math.nan
    kd, vd = k.cuda(), v.cuda()
    ops.rope_kv_write_fp4(qkv.cuda(), pos.cuda(), cs.cuda(), kd, vd, slots.cuda(), hq, hk, d, 0)
    ops.rope_kv_write_fp4(qkv, pos, cs, k, v, slots, hq, hk, d, 0)
    assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v)
    kr, vr = ops.kv_fp4_read(kd, vd, slots.cuda(), d)
    assert torch.isfinite(kr).all() and torch.isfinite(vr).all()
    assert (kr[0] == 0).all() and (kr[3] == 2688).all()


@pytest.mark.parametrize("hq,hk,d,rot", [(32, 8, 128, 128), (16, 2, 256, 64), (4, 2, 64, 64), (7, 1, 128, 96), (3, 3, 64, 0),
                                         (5, 3, 256, 256), (4, 1, 256, 0), (1, 5, 128, 32), (4, 2, 128, 24)])
@pytest.mark.parametrize("T", [599, 1199, 2503])
def test_write_many_tokens(hq, hk, d, rot, T):
    """Tokens that share warps, some of them not cached, positions outside the table, and rows of any stride."""
    qkv, pos, cs, slots, k, v = write_case(T, hq, hk, d, rot, seed=T + d, pad=8 * (hq % 2))
    slots[::7], slots[5], slots[T - 1] = -1, 1 << 40, -(1 << 40)
    pos[11], pos[12] = -3, 512
    want_pos = torch.where((pos < 0) | (pos >= 512), 0, pos)  # positions outside the table read its first row
    kd, vd = k.cuda(), v.cuda()
    q = ops.rope_kv_write_fp4(qkv.cuda(), pos.cuda(), cs.cuda(), kd, vd, slots.cuda(), hq, hk, d, rot, 0.75, 2.0)
    want = ops.rope_kv_write_fp4(qkv, want_pos, cs, k, v, slots, hq, hk, d, rot, 0.75, 2.0)
    assert torch.equal(q.cpu(), want)
    assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v)
    kr, vr = ops.kv_fp4_read(kd, vd, slots.cuda(), d, 0.75, 2.0)
    kw, vw = ops.kv_fp4_read(k, v, slots, d, 0.75, 2.0)
    assert torch.equal(kr.cpu(), kw.bfloat16()) and torch.equal(vr.cpu(), vw.bfloat16())


@pytest.mark.parametrize("T", [40, 1280])
def test_write_values_on_and_beside_the_ties(T):
    """Every scale mantissa, values on each tie between two codes and the nearest bf16 values on both sides of it."""
    hq, hk, d = 2, 1, 128
    qkv, pos, cs, slots, k, v = write_case(T, hq, hk, d, 0, seed=6)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    for t in range(T):
        for b in range(8):
            s = (8 + b) / 8.0 * 2.0 ** (t % 40 - 20 if t % 40 > 14 else t % 40 - 6)
            s = max(s, 2.0 ** -8)
            tie = (ties * s).bfloat16()
            beside = torch.cat((tie.view(torch.int16) + 1, tie.view(torch.int16) - 1)).view(torch.bfloat16)
            x = torch.cat((tie, beside))[torch.randperm(21, generator=torch.Generator().manual_seed(t * 8 + b))[:15]]
            x = torch.cat((torch.tensor([6.0 * s]).bfloat16(), x)) * (1 if t % 2 else -1)
            qkv[t, hq * d + 16 * b: hq * d + 16 * b + 16] = x
            qkv[t, (hq + 1) * d + 16 * b: (hq + 1) * d + 16 * b + 16] = x.flip(0)
    kd, vd = k.cuda(), v.cuda()
    ops.rope_kv_write_fp4(qkv.cuda(), pos.cuda(), cs.cuda(), kd, vd, slots.cuda(), hq, hk, d, 0, 1.0, 0.5)
    ops.rope_kv_write_fp4(qkv, pos, cs, k, v, slots, hq, hk, d, 0, 1.0, 0.5)
    assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v)


@pytest.mark.parametrize("T", [3, 1300])
def test_write_extremes_and_an_odd_table_start(T):
    """Infinities and NaN in some blocks only; a cosine table that starts on 4 bytes."""
    hq, hk, d = 2, 2, 128
    qkv, pos, cs, slots, k, v = write_case(T, hq, hk, d, 64, seed=8)
    qkv[::3, 5::16] = math.inf
    qkv[1::3, 9::32] = -math.inf
    qkv[2::3, 700::40] = math.nan
    buf = torch.zeros(cs.numel() + 1, device="cuda")
    buf[1:] = cs.flatten().cuda()
    odd = buf[1:].view(cs.shape)
    kd, vd = k.cuda(), v.cuda()
    q = ops.rope_kv_write_fp4(qkv.cuda(), pos.cuda(), odd, kd, vd, slots.cuda(), hq, hk, d, 64)
    want = ops.rope_kv_write_fp4(qkv, pos, cs, k, v, slots, hq, hk, d, 64)
    assert torch.equal(q.cpu().isnan(), want.isnan()) and torch.equal(q.cpu().nan_to_num(), want.nan_to_num())
    assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v)


def test_write_refusals():
    qkv, pos, cs, slots, k, v = (t.cuda() for t in write_case(4, 4, 2, 64, 64))

    def call(**kw):
        a = dict(qkv=qkv, pos=pos, cs=cs, k=k, v=v, slots=slots, hq=4, hk=2, d=64, rot=64, gk=1.0, q_out=None)
        a.update(kw)
        ops.rope_kv_write_fp4(a["qkv"], a["pos"], a["cs"], a["k"], a["v"], a["slots"], a["hq"], a["hk"], a["d"], a["rot"],
                              a["gk"], 1.0, a["q_out"])

    call()
    for kw in (dict(qkv=qkv.half()), dict(qkv=qkv[:, :-64]), dict(pos=pos[:-1]), dict(pos=pos.int()), dict(cs=cs[:, :-2]),
               dict(k=k[:, :1]), dict(slots=slots.int()), dict(hk=4), dict(d=48), dict(rot=63, cs=cs[:, :63]),
               dict(gk=-1.0), dict(q_out=qkv[:, :256]), dict(q_out=torch.empty(4, 128, dtype=torch.bfloat16, device="cuda"))):
        with pytest.raises((RuntimeError, ValueError)):
            call(**kw)


# ----------------------------------------------------------------------------------------------- page copies
@pytest.mark.parametrize("n", [0, 1, 7])
def test_copy_pages(n):
    g = torch.Generator().manual_seed(n)
    caches = [torch.randint(0, 256, ops.kv_fp4_cache_shape(20, 2, d), generator=g, dtype=torch.uint8) for d in (64, 128, 256)]
    caches += [torch.randn(20, 3, 64, 64, generator=g).bfloat16(), torch.randn(16, 4, generator=g)]
    caches += [torch.randint(0, 256, (20, 16), generator=g, dtype=torch.uint8) for _ in range(130)]  # more than a launch takes
    ids = torch.randperm(16, generator=g)
    src, dst = ids[:n].contiguous(), ids[n:2 * n].contiguous()
    if n > 3:
        src[0], dst[1], src[2], dst[3] = -1, -5, 20, 1 << 40
    dev = [c.cuda() for c in caches]
    ops.copy_kv_pages(dev, src.cuda(), dst.cuda())
    ops.copy_kv_pages(caches, src, dst)
    for a, b in zip(dev, caches):
        assert torch.equal(a.cpu(), b)


def test_copy_refusals():
    c = torch.zeros(8, 64, dtype=torch.uint8, device="cuda")
    ids = torch.arange(2, device="cuda")
    ops.copy_kv_pages([c], ids, ids + 2)
    for caches, src, dst in (([c.t()], ids, ids), ([c], ids.int(), ids), ([c], ids, ids[:1]), ([c], ids.cpu(), ids),
                             ([c, c.cpu()], ids, ids), ([torch.zeros(8, 3, dtype=torch.uint8, device="cuda")], ids, ids)):
        with pytest.raises(RuntimeError):
            ops.copy_kv_pages(caches, src, dst)
