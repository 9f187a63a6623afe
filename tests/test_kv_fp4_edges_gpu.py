"""The 4-bit KV cache on the GPU, at the edges of its plans: cut units, scratch, strides, streams, refusals."""
import math

import pytest
import torch

from test_kv_fp4_gpu import attend, case, check
from vllm_suffix_hybrid_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q,seq", [(2000, 512), (5120, 576), (1500, 700), (2304, 513)])
@pytest.mark.parametrize("hq,d", [(1, 128), (2, 128), (1, 256), (1, 64)])
def test_more_new_tokens_than_keys_over_many_runs(q, seq, hq, d):
    """Rows before the first key weigh nothing: the few units that see keys are cut, every cut has its partial, and
    nothing of an earlier call's partials is merged."""
    cols = None if d == 128 else 4000  # a wide table says that the work may be large
    attend(case((700,), (9000,), 8, 1, d, seed=40, gain=4.0, cols=cols))  # leaves partials of every run behind
    c = case((q,), (seq,), hq, 1, d, seed=41, cols=cols)
    got = attend(c)
    check(c, got)
    assert (got[: q - seq] == 0).all()
    assert torch.equal(got, attend(c))


DECODE, VERIFY = ((1,) * 5, (7000,) * 5), ((2,) * 4, (9000,) * 4)
PROMPT, PROMPTS = ((300,), (9000,)), ((90, 200), (5000, 700))


@pytest.mark.parametrize("shapes", [(DECODE, VERIFY), (PROMPT, PROMPTS), (DECODE, PROMPT)])
def test_branches_of_one_graph_do_not_disturb_each_other(shapes):
    """Calls with cut units on two streams of one capture: each branch has partials and tickets of its own."""
    cases = [case(q, s, 8, 2, 128, seed=50 + i) for i, (q, s) in enumerate(shapes)]
    dev = [{n: c[n].cuda() for n in ("q", "k", "v", "bt", "seqs", "qs")} for c in cases]
    outs = [torch.empty_like(d["q"]) for d in dev]

    def call(i):
        c, d = cases[i], dev[i]
        for _ in range(3):
            ops.paged_attention_fp4(outs[i], d["q"], d["k"], d["v"], d["bt"], d["seqs"], d["qs"], 8, 128, c["scale"],
                                    c["max_q"], c["gk"], c["gv"])

    want = []
    for i in range(2):
        call(i)
        check(cases[i], outs[i])
        want.append(outs[i].clone())
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call(1)
        call(0)
        torch.cuda.current_stream().wait_stream(side)
    for _ in range(20):
        for o in outs:
            o.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


@pytest.mark.parametrize("length", [2 ** 31 - 64, 2 ** 31, 2 ** 40])
def test_lengths_at_and_beyond_the_widest_table(length):
    """2^31 positions and more: a length is clipped below 2^31, not wrapped.  Every key is block 0's zero and every value
    a one, so sums of fewer than 2^24 of them are exact and the result is 1 but for the merges' roundings."""
    k = torch.zeros(ops.kv_fp4_cache_shape(1, 1, 64), dtype=torch.uint8, device="cuda")
    v = k.clone()
    v[..., :32 * 64] = 0x22  # e2m1 1.0, twice
    v[..., 32 * 64:] = 0x38  # e4m3 1.0
    q = torch.ones(1, 8 * 64, dtype=torch.bfloat16, device="cuda")
    out = torch.full_like(q, math.nan)
    bt = torch.zeros(1, 2 ** 25, dtype=torch.int32, device="cuda")
    ops.paged_attention_fp4(out, q, k, v, bt, torch.tensor([length], device="cuda"), torch.tensor([0, 1], device="cuda"), 8,
                            64, 0.125, 1)
    assert (out == 1).all()


@pytest.mark.parametrize("off", [1, 2, 4, 8])
@pytest.mark.parametrize("which", [0, 1])
def test_caches_that_start_off_16_bytes_are_refused(off, which):
    """A contiguous view into a larger buffer may start anywhere; every entry point says so before it launches."""
    shape = ops.kv_fp4_cache_shape(2, 1, 64)
    n = math.prod(shape)
    caches = [torch.zeros(shape, dtype=torch.uint8, device="cuda") for _ in range(2)]
    caches[which] = torch.zeros(n + 16, dtype=torch.uint8, device="cuda")[off:off + n].view(shape)
    one = torch.zeros(1, dtype=torch.long, device="cuda")
    q = torch.zeros(1, 3 * 64, dtype=torch.bfloat16, device="cuda")
    cs = torch.zeros(4, 64, device="cuda")
    for call in (lambda: ops.kv_fp4_read(*caches, one, 64),
                 lambda: ops.rope_kv_write_fp4(q, one, cs, *caches, one, 1, 1, 64),
                 lambda: ops.paged_attention_fp4(torch.empty_like(q), q, *caches, one[None].int(), one,
                                                 torch.tensor([0, 1], device="cuda"), 1, 64, 0.1, 1),
                 lambda: ops.copy_kv_pages(caches, one, one + 1)):
        with pytest.raises(RuntimeError, match="aligned"):
            call()


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_caches_on_two_devices_are_refused():
    shape = ops.kv_fp4_cache_shape(2, 1, 64)
    caches = [torch.zeros(shape, dtype=torch.uint8, device=f"cuda:{i}") for i in range(2)]
    one = torch.zeros(1, dtype=torch.long, device="cuda:0")
    q = torch.zeros(1, 3 * 64, dtype=torch.bfloat16, device="cuda:0")
    cs = torch.zeros(4, 64, device="cuda:0")
    for call in (lambda: ops.kv_fp4_read(*caches, one, 64),
                 lambda: ops.rope_kv_write_fp4(q, one, cs, *caches, one, 1, 1, 64),
                 lambda: ops.paged_attention_fp4(torch.empty_like(q), q, *caches, one[None].int(), one,
                                                 torch.tensor([0, 1], device="cuda:0"), 1, 64, 0.1, 1)):
        with pytest.raises(RuntimeError, match="one device"):
            call()


@pytest.mark.parametrize("bad", [0.0, -1.0, math.inf, math.nan, 1e300, 1e-300, 1e-40])
def test_scales_that_fp32_cannot_hold_are_refused(bad):
    """An infinite scale made every cached value a zero or a NaN, and one below fp32's range saturated every code."""
    cache = torch.zeros(ops.kv_fp4_cache_shape(2, 1, 64), dtype=torch.uint8, device="cuda")
    one = torch.zeros(1, dtype=torch.long, device="cuda")
    q = torch.zeros(1, 3 * 64, dtype=torch.bfloat16, device="cuda")
    cs = torch.zeros(4, 64, device="cuda")
    for gk, gv in ((bad, 1.0), (1.0, bad)):
        for call in (lambda: ops.kv_fp4_read(cache, cache, one, 64, gk, gv),
                     lambda: ops.rope_kv_write_fp4(q, one, cs, cache, cache, one, 1, 1, 64, 64, gk, gv),
                     lambda: ops.paged_attention_fp4(torch.empty_like(q), q, cache, cache, one[None].int(), one,
                                                     torch.tensor([0, 1], device="cuda"), 1, 64, 0.1, 1, gk, gv)):
            with pytest.raises(RuntimeError, match="scales"):
                call()


def test_partials_take_what_the_kernel_writes():
    """Two partials a run of each query tile: one tile of 256 dimensions is as much as two of 128."""
    import ctypes

    from vllm_suffix_hybrid_b200 import _C

    size = ctypes.CDLL(_C.__file__).sh_paged_attention_fp4_tc_workspace
    size.restype, size.argtypes = ctypes.c_int64, [ctypes.c_int]
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    torch.zeros(1, device="cuda")  # the function asks for the current device
    for d, tiles in ((64, 2), (128, 2), (256, 1)):
        partials = sms * 2 * tiles * (d + 2) * 128
        assert partials < size(d) <= partials + sms * 16


def test_the_error_word():
    """It stays zero where no wait runs out, and has to be an int32 on the caches' device."""
    c = case((300, 200), (4000, 200), 8, 2, 128, seed=60)
    dev = {n: c[n].cuda() for n in ("q", "k", "v", "bt", "seqs", "qs")}
    out = torch.empty_like(dev["q"])

    def call(err):
        ops.paged_attention_fp4(out, dev["q"], dev["k"], dev["v"], dev["bt"], dev["seqs"], dev["qs"], 8, 128, c["scale"],
                                c["max_q"], c["gk"], c["gv"], err=err)

    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    call(err)
    check(c, out)
    assert err.item() == 0
    for bad in (err.long(), err.cpu(), err[:0]):
        with pytest.raises(RuntimeError, match="err must be"):
            call(bad)


# ----------------------------------------------------------------------------------------------- plans of many rows
@pytest.mark.parametrize("hq,hk,d", [(8, 2, 128), (8, 1, 256), (12, 3, 64)])
def test_many_strided_rows_and_a_strided_table(hq, hk, d):
    """Whole and cut units whose rows are columns of wider tensors, over a table with spare columns."""
    c = case((300, 41, 0, 700), (5000, 41, 7, 900), hq, hk, d, seed=70 + d, cols=4000)
    T = c["q"].shape[0]
    wide = torch.randn(T, 2 * hq * d + 64, device="cuda").bfloat16()
    wide[:, 64:64 + hq * d] = c["q"].cuda()
    outw = torch.zeros(T, hq * d + 24, dtype=torch.bfloat16, device="cuda")
    bt = torch.randint(0, 1 << 30, (4, 4007), dtype=torch.int32)
    bt[:, :4000] = c["bt"]
    got = outw[:, 16:16 + hq * d]
    ops.paged_attention_fp4(got, wide[:, 64:64 + hq * d], c["k"].cuda(), c["v"].cuda(), bt.cuda()[:, :4000],
                            c["seqs"].cuda(), c["qs"].cuda(), hq, d, c["scale"], 700, c["gk"], c["gv"])
    check(c, got)
    assert (outw[:, :16] == 0).all() and (outw[:, 16 + hq * d:] == 0).all()


@pytest.mark.parametrize("hq,hk,d", [(8, 2, 128), (8, 1, 256), (8, 2, 64)])
def test_a_captured_prompt_follows_its_lengths(hq, hk, d):
    """The tensor-core kernel and its merge under capture: lengths and tables are read at replay."""
    c = case((300, 130), (5000, 4000), hq, hk, d, seed=80 + d, cols=4000)
    dev = {n: c[n].cuda() for n in ("k", "v", "bt", "seqs", "qs", "q")}
    out = torch.empty_like(dev["q"])

    def call():
        for _ in range(2):
            ops.paged_attention_fp4(out, dev["q"], dev["k"], dev["v"], dev["bt"], dev["seqs"], dev["qs"], hq, d, c["scale"],
                                    300, c["gk"], c["gv"])

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for seqs in ((5000, 4000), (300, 3968), (4999, 130), (64, 200)):
        c["seqs"] = torch.tensor(seqs)
        dev["seqs"].copy_(c["seqs"])
        for _ in range(2):
            out.fill_(math.nan)
            graph.replay()
        torch.cuda.synchronize()
        check(c, out)


def test_prompts_on_two_streams_do_not_disturb_each_other():
    a, b = case((500, 60), (3000, 6000), 8, 2, 128, seed=90), case((400,), (5000,), 8, 1, 256, seed=91, cols=4000)
    ra, rb = attend(a), attend(b)
    check(a, ra)
    check(b, rb)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            got.append(attend((a, b)[i % 2]))
    torch.cuda.synchronize()
    for i, r in enumerate(got):
        assert torch.equal(r, (ra, rb)[i % 2])


@pytest.mark.parametrize("hq,hk,d", [(8, 2, 128), (8, 1, 256), (8, 2, 64)])
def test_bad_block_ids_under_many_rows_stay_in_bounds(hq, hk, d):
    """Ids outside the cache read block 0, whatever it holds; only the rows that use them are affected."""
    c = case((200, 150), (3000, 2000), hq, hk, d, seed=100 + d, cols=4000)
    c["bt"][0, 1], c["bt"][0, 2], c["bt"][0, 46] = 1 << 30, -7, c["k"].shape[0]
    got = attend(c)
    c["bt"][0, 1:3] = c["bt"][0, 46] = 0
    same = attend(c)
    assert torch.equal(got.view(torch.int16), same.view(torch.int16))
    check(dict(c, q=c["q"][200:], bt=c["bt"][1:], seqs=c["seqs"][1:], qs=torch.tensor([0, 150])), got[200:])


# ----------------------------------------------------------------------------------------------- many requests
@pytest.mark.parametrize("hq,hk,d", [(4, 2, 128), (2, 1, 256), (2, 2, 64)])
@pytest.mark.parametrize("B", [129, 200, 256, 300, 777])
def test_more_requests_than_threads(hq, hk, d, B):
    """A CTA's threads look at the requests in several passes; runs begin in every one of them."""
    g = torch.Generator().manual_seed(B)
    seqs = torch.randint(0, 500, (B,), generator=g).tolist()
    q = torch.randint(0, 4, (B,), generator=g).tolist()
    q[:90] = [0] * 90 if B > 300 else q[:90]  # a first pass that is almost empty
    q = [min(a, s) if s else a for a, s in zip(q, seqs)]
    c = case(q, seqs, hq, hk, d, seed=B + d)
    got = attend(c)
    check(c, got)
    assert torch.equal(got, attend(c))


@pytest.mark.parametrize("hq,hk,d", [(4, 2, 128), (2, 1, 256), (2, 2, 64)])
def test_many_requests_of_many_rows(hq, hk, d):
    """The same for the tensor-core kernel, whose CTAs have 416 to 512 threads."""
    g = torch.Generator().manual_seed(7)
    seqs = torch.randint(1, 300, (600,), generator=g).tolist()
    q = [min(s, 3) for s in seqs]
    q[550], seqs[550] = 200, 700
    c = case(q, seqs, hq, hk, d, seed=110 + d, cols=4000)
    check(c, attend(c))


@pytest.mark.parametrize("d,hk", [(64, 8), (128, 8), (256, 4)])
def test_pages_beyond_four_gigabytes(d, hk):
    """Blocks whose bytes start beyond 2^32: written, read, attended and copied as those of a small cache, bit for bit."""
    hq, T = 2 * hk, 700
    page = hk * ops.kv_fp4_cache_shape(1, hk, d)[2]
    base = 2 ** 32 // page + 1
    g = torch.Generator(device="cuda").manual_seed(d)
    qkv = torch.randn(T, (hq + 2 * hk) * d, device="cuda", generator=g).bfloat16()
    pos = torch.arange(T, device="cuda")
    cs = ops.ref.rope_cos_sin(T, d, 10000.0).cuda()
    got = []
    for first in (1, base):
        caches = [torch.zeros(ops.kv_fp4_cache_shape(first + 24, hk, d), dtype=torch.uint8, device="cuda") for _ in range(2)]
        assert first == 1 or caches[0][first:].data_ptr() - caches[0].data_ptr() > 2 ** 32
        bt = first + torch.randperm(11, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
        slots = bt[pos // 64] * 64 + pos % 64
        q = ops.rope_kv_write_fp4(qkv, pos, cs, *caches, slots, hq, hk, d)
        rows = ops.kv_fp4_read(*caches, slots, d)
        few = ops.rope_kv_write_fp4(qkv[:5], pos[:5], cs, *caches, slots[:5], hq, hk, d)  # the kernel for few tokens
        again = ops.kv_fp4_read(*caches, slots, d)
        ops.copy_kv_pages(caches, bt, bt + 12)
        copied = ops.kv_fp4_read(*caches, slots + 12 * 64, d)
        outs = []
        for n in (1, 6, T):
            out = torch.full((n, hq * d), math.nan, dtype=torch.bfloat16, device="cuda")
            for table in (bt, bt + 12):
                wide = torch.zeros(1, 4000, dtype=torch.int32, device="cuda")
                wide[0, :11] = table
                ops.paged_attention_fp4(out, q[-n:], *caches, wide, torch.tensor([T], device="cuda"),
                                        torch.tensor([0, n], device="cuda"), hq, d, d ** -0.5, n)
                outs.append(out.clone())
        assert torch.isfinite(outs[-1]).all() and (outs[-1] != 0).any()
        got.append([q, few, *rows, *again, *copied, *outs])
        del caches
    for a, b in zip(*got):
        assert torch.equal(a, b)
