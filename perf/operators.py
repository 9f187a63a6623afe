"""The operators of the 4-bit paged KV cache, as they are measured.

Three operators, each in its plain form (elementary torch operations in 32 bits) and, with ``own`` set, through the
framework's entry points:

* ``write``  -- RoPE of the new tokens' queries and keys, NVFP4 quantisation of keys and values into their cache
  pages, and the cached rows read back as the values that they stand for;
* ``attend`` -- causal GQA attention of the new tokens over the 4-bit pages (decode, verify window, prefill);
* ``copy``   -- page copies in every layer's cache (fork of a sequence, compaction of the pool).

A cache tensor is uint8 [num_blocks, kv_heads, 64 * (D/2 + D/16)]: per (block, head) the 64 tokens' codes (two e2m1
codes a byte, even dimension in the low nibble), then their e4m3 scales, one per 16 dimensions.
"""
import math

import torch

own = False

BLOCK = 64
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------------------------------------- cases
def listed():
    llama = dict(hq=32, hk=8, d=128, rot=128)  # the 8B dense decoder's attention
    hybrid = dict(hq=16, hk=2, d=256, rot=64)  # the hybrid model's gated attention, partial rotary
    return [
        # one decoding request appends its token: launch latency
        dict(name="write-decode-1", op="write", tokens=1, **llama),
        # a verify step of the wide-head model, an odd number of tokens
        dict(name="write-verify-389", op="write", tokens=389, **hybrid),
        # a full prefill batch
        dict(name="write-prefill-16384", op="write", tokens=16384, **llama),
        # a single request with a short history: latency
        dict(name="decode-1x1000", op="attend", batch=1, q=1, ctx=1000, **llama),
        # the serving batch, plain decode at mixed lengths
        dict(name="decode-64x2048", op="attend", batch=64, q=1, ctx=2048, **llama),
        # a speculative verify step (five drafts) at mixed lengths
        dict(name="verify-32x8191", op="attend", batch=32, q=6, ctx=8191, **llama),
        # few very long requests: the cache read alone
        dict(name="decode-8x131072", op="attend", batch=8, q=1, ctx=131072, **llama),
        # 256-wide heads, eight query heads a key head
        dict(name="decode-24x4000", op="attend", batch=24, q=1, ctx=4000, **hybrid),
        # one whole prompt
        dict(name="prefill-8192", op="attend", batch=1, q=8192, ctx=8192, **llama),
        # the next chunk of a long prompt
        dict(name="chunk-2000x32768", op="attend", batch=1, q=2000, ctx=32768, **llama),
        # fork of one sequence: its last, partial page in all layers
        dict(name="copy-1", op="copy", layers=32, blocks=256, pages=1, hk=8, d=128),
        # compaction of a large pool
        dict(name="copy-1023", op="copy", layers=32, blocks=2500, pages=1023, hk=8, d=128),
    ]


def _log(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    n = min(max(n, lo), hi)
    return n - 1 if n % 1024 == 0 and n > 1024 else n


HEADS = (dict(hq=32, hk=8, d=128, rot=128), dict(hq=16, hk=2, d=256, rot=64), dict(hq=8, hk=2, d=64, rot=64),
         dict(hq=8, hk=8, d=128, rot=128), dict(hq=4, hk=1, d=128, rot=64), dict(hq=28, hk=4, d=128, rot=128))


def draw(rng):
    """A case of the listed ranges: any head layout, token counts and lengths over their whole ranges."""
    op = rng.choice(("write", "attend", "attend", "attend", "copy"))
    heads = dict(rng.choice(HEADS))
    if op == "write":
        return dict(op=op, tokens=_log(rng, 1, 16384), **heads)
    if op == "copy":
        blocks = _log(rng, 64, 2500)
        return dict(op=op, layers=rng.choice((1, 2, 13, 32)), blocks=blocks, pages=_log(rng, 1, max(1, blocks // 3)),
                    hk=heads["hk"], d=heads["d"])
    kind = rng.choice(("decode", "verify", "prefill", "chunk"))
    if kind == "decode":
        batch = _log(rng, 1, 256)
        return dict(op=op, batch=batch, q=1, ctx=_log(rng, 1, min(131072, 524288 // batch)), **heads)
    if kind == "verify":
        batch, q = _log(rng, 1, 64), rng.randint(2, 9)
        return dict(op=op, batch=batch, q=q, ctx=_log(rng, q, min(65536, 262144 // batch)), **heads)
    if kind == "prefill":
        batch = rng.choice((1, 1, 2, 5, 8))
        q = _log(rng, 17, 8192 // batch)
        return dict(op=op, batch=batch, q=q, ctx=q, **heads)
    q = _log(rng, 17, 2000)
    return dict(op=op, batch=1, q=q, ctx=q + _log(rng, 64, 30000), **heads)


def _lengths(case):
    """(new tokens, length with them) of each request: the first has the case's own, the others are shorter."""
    out = []
    for i in range(case["batch"]):
        cut = (i * 977) % (case["ctx"] // 2 + 1)
        n = case["ctx"] - cut
        q = min(case["q"], n)
        if case["q"] == case["ctx"]:
            q = n  # whole prompts
        out.append((q, n))
    return out


def page_bytes(d):
    return BLOCK * (d // 2 + d // 16)


def work(case):
    if case["op"] == "copy":
        return {"bytes": 2 * case["pages"] * case["layers"] * 2 * case["hk"] * page_bytes(case["d"]), "flops": 0}
    hq, hk, d = case["hq"], case["hk"], case["d"]
    row = d // 2 + d // 16
    if case["op"] == "write":
        t = case["tokens"]
        # the projection rows and the rotary rows read, the queries, the cache rows and the values read back written
        return {"bytes": t * (2 * (hq + 2 * hk) * d + 4 * case["rot"] + 16 + 2 * hq * d + 2 * hk * row + 4 * hk * d),
                "flops": t * (3 * (hq + hk) * case["rot"] + 8 * hk * d)}
    q = sum(a for a, _ in _lengths(case))
    keys = sum(n for _, n in _lengths(case))
    pairs = sum(a * n - a * (a - 1) // 2 for a, n in _lengths(case))
    return {"bytes": 4 * q * hq * d + 2 * keys * hk * row, "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------------------------------------------- NVFP4, plain
def _round_e4m3(x):
    """Nearest e4m3 value (ties to even) of 2^-9 <= x <= 448, as fp32."""
    e = torch.floor(torch.log2(x)).clamp(min=-6.0)
    e = torch.where(torch.exp2(e) > x, e - 1, e).clamp(min=-6.0)
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def _e4m3_byte(s):
    """Bits of an e4m3 value >= 0 given exactly in fp32."""
    e = torch.floor(torch.log2(s.clamp(min=2.0 ** -9))).clamp(min=-6.0)
    m = torch.where(s < 2.0 ** -6, s * 2.0 ** 9, (s * torch.exp2(-e) - 1) * 8)
    return torch.where(s < 2.0 ** -6, m, (e + 7) * 8 + m).to(torch.uint8)


def _code(y):
    """Nearest e2m1 code (ties to the even code) of y, saturating at 6; bit 3 is the sign."""
    a = y.abs()
    c = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    return c.to(torch.uint8) + 8 * torch.signbit(y).to(torch.uint8)


def _quantise(x):
    """x fp32 [..., D] -> (codes uint8 [..., D], block scales fp32 [..., D/16])."""
    b = x.unflatten(-1, (-1, 16))
    six = torch.full((), 6.0, device=x.device)  # a tensor: division by a Python number multiplies by its reciprocal
    s = _round_e4m3((b.abs().amax(-1) / six).clamp(2.0 ** -9, 448.0))
    return _code(b / s[..., None]).flatten(-2), s


def _pack(codes, s):
    """Rows' bytes: (codes [..., D/2], scales [..., D/16]) uint8."""
    return codes[..., 0::2] + 16 * codes[..., 1::2], _e4m3_byte(s)


def _unpack(codes, scales, scale):
    """Packed codes [..., D/2] and scale bytes [..., D/16] -> fp32 values [..., D]."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float32, device=codes.device)
    v = torch.stack((table[(codes & 15).long()], table[(codes >> 4).long()]), -1).flatten(-2)
    e, m = (scales >> 3 & 15).float(), (scales & 7).float()
    s = torch.where(e == 0, m * 2.0 ** -9, torch.exp2(e - 7) * (1 + m / 8))
    return (v.unflatten(-1, (-1, 16)) * s[..., None]).flatten(-2) * scale


# ------------------------------------------------------------------------------------------------- inputs
def _values(shape, gen, spread):
    """Projection-like values: normal, with a few channels several times the others."""
    x = torch.randn(shape, generator=gen, device="cuda")
    gain = torch.exp(spread * torch.randn(shape[-1], generator=gen, device="cuda"))
    return x * gain


def _cache(blocks, hk, d, gen, spread):
    cache = torch.empty(blocks, hk, page_bytes(d), dtype=torch.uint8, device="cuda")
    split = BLOCK * d // 2
    for lo in range(0, blocks, 1024):
        n = min(1024, blocks - lo)
        codes, scales = _pack(*_quantise(_values((n, hk, BLOCK, d), gen, spread)))
        cache[lo:lo + n, :, :split] = codes.flatten(-2)
        cache[lo:lo + n, :, split:] = scales.flatten(-2)
    return cache


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] == "copy":
        shape = (2 * case["layers"], case["blocks"], case["hk"], page_bytes(case["d"]))
        s["pool"] = torch.randint(0, 0x70, shape, generator=gen, device="cuda", dtype=torch.uint8)
        ids = torch.randperm(case["blocks"] - 1, generator=gen, device="cuda") + 1
        s["src"], s["dst"] = ids[: case["pages"]].contiguous(), ids[case["pages"]: 2 * case["pages"]].contiguous()
        s["caches"] = list(s["pool"].unbind(0))  # one tensor per layer and side, as an engine holds them
        return s
    hq, hk, d, rot = case["hq"], case["hk"], case["d"], case["rot"]
    if case["op"] == "write":
        t = case["tokens"]
        s["qkv"] = _values((t, (hq + 2 * hk) * d), gen, 0.5).bfloat16()
        s["positions"] = torch.randint(0, 32768, (t,), generator=gen, device="cuda")
        inv = 1.0 / (500000.0 ** (torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot))
        ang = torch.arange(32768, dtype=torch.float64, device="cuda")[:, None] * inv
        s["cos_sin"] = torch.cat((ang.cos(), ang.sin()), 1).float()
        blocks = t // BLOCK + 3
        slots = torch.randperm((blocks - 1) * BLOCK, generator=gen, device="cuda")[:t] + BLOCK
        if t > 8:
            slots[::t // 4] = -1  # padded rows of a batch bucket: nothing cached
        s["slots"] = slots
        s["k_cache"] = torch.zeros(blocks, hk, page_bytes(d), dtype=torch.uint8, device="cuda")
        s["v_cache"] = torch.zeros_like(s["k_cache"])
        s["k_scale"], s["v_scale"] = 1.0, 0.5
        return s
    lens = _lengths(case)
    pages = [-(-n // BLOCK) for _, n in lens]
    blocks = sum(pages) + 1
    ids = (torch.randperm(blocks - 1, generator=gen, device="cuda") + 1).to(torch.int32)
    at = torch.arange(max(pages), device="cuda")[None, :] + torch.tensor([0] + pages[:-1], device="cuda").cumsum(0)[:, None]
    live = torch.arange(max(pages), device="cuda")[None, :] < torch.tensor(pages, device="cuda")[:, None]
    s["block_tables"] = torch.where(live, ids[at.clamp(max=blocks - 2)], 0).to(torch.int32)
    s["seq_lens"] = torch.tensor([n for _, n in lens], device="cuda")
    s["q_start"] = torch.tensor([0] + [a for a, _ in lens], device="cuda").cumsum(0)
    s["max_q"] = max(a for a, _ in lens)
    s["q"] = _values((sum(a for a, _ in lens), hq * d), gen, 0.3).bfloat16()
    s["k_cache"], s["v_cache"] = _cache(blocks, hk, d, gen, 0.5), _cache(blocks, hk, d, gen, 0.2)
    s["scale"], s["k_scale"], s["v_scale"] = 1.0 / math.sqrt(d), 0.75, 0.5
    return s


# ------------------------------------------------------------------------------------------------- one pass
def run(s):
    if s["op"] == "copy":
        return _copy_own(s) if own else _copy_plain(s)
    if s["op"] == "write":
        return _write_own(s) if own else _write_plain(s)
    return _attend_own(s) if own else _attend_plain(s)


def _copy_own(s):
    from vllm_suffix_hybrid_b200 import ops

    ops.copy_kv_pages(s["caches"], s["src"], s["dst"])
    return s["pool"]


def _copy_plain(s):
    s["pool"][:, s["dst"]] = s["pool"][:, s["src"]]
    return s["pool"]


def _write_own(s):
    from vllm_suffix_hybrid_b200 import ops

    q = ops.rope_kv_write_fp4(s["qkv"], s["positions"], s["cos_sin"], s["k_cache"], s["v_cache"], s["slots"], s["hq"],
                              s["hk"], s["d"], s["rot"], s["k_scale"], s["v_scale"])
    k, v = ops.kv_fp4_read(s["k_cache"], s["v_cache"], s["slots"], s["d"], s["k_scale"], s["v_scale"])
    return q, k, v


def _rope(x, cos, sin):
    half = cos.shape[-1]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]), -1)


def _store(cache, slots, x, scale, d):
    """Quantises rows x [T, hk, D] into their slots (a slot below 0 is dropped)."""
    codes, scales = _pack(*_quantise(x * (1.0 / scale)))
    keep = slots >= 0
    blk, off = slots[keep] // BLOCK, slots[keep] % BLOCK
    split = BLOCK * d // 2
    cache[:, :, :split].unflatten(-1, (BLOCK, -1))[blk, :, off] = codes[keep]
    cache[:, :, split:].unflatten(-1, (BLOCK, -1))[blk, :, off] = scales[keep]


def _load(cache, slots, scale, d):
    """The values of the slots' rows [T, hk, D] in bf16; zeros for a slot below 0."""
    at = slots.clamp(min=0)
    blk, off = at // BLOCK, at % BLOCK
    split = BLOCK * d // 2
    x = _unpack(cache[:, :, :split].unflatten(-1, (BLOCK, -1))[blk, :, off],
                cache[:, :, split:].unflatten(-1, (BLOCK, -1))[blk, :, off], scale)
    return torch.where((slots >= 0)[:, None, None], x, 0.0).bfloat16()


def _write_plain(s):
    hq, hk, d = s["hq"], s["hk"], s["d"]
    x = s["qkv"].float().unflatten(-1, (-1, d))
    cos, sin = s["cos_sin"][s["positions"]][:, None].chunk(2, -1)
    q, k, v = _rope(x[:, :hq], cos, sin), _rope(x[:, hq:hq + hk], cos, sin), x[:, hq + hk:hq + 2 * hk]
    _store(s["k_cache"], s["slots"], k, s["k_scale"], d)
    _store(s["v_cache"], s["slots"], v, s["v_scale"], d)
    return (q.flatten(1).bfloat16(), _load(s["k_cache"], s["slots"], s["k_scale"], d),
            _load(s["v_cache"], s["slots"], s["v_scale"], d))


def _attend_own(s):
    from vllm_suffix_hybrid_b200 import ops

    out = torch.empty_like(s["q"])
    ops.paged_attention_fp4(out, s["q"], s["k_cache"], s["v_cache"], s["block_tables"], s["seq_lens"], s["q_start"],
                            s["hq"], s["d"], s["scale"], s["max_q"], s["k_scale"], s["v_scale"])
    return out


def _gather(cache, tables, scale, d):
    """The requests' keys or values, fp32 [B, hk, pages * 64, D]."""
    pages = cache[tables.long()]
    split = BLOCK * d // 2
    x = _unpack(pages[..., :split].unflatten(-1, (BLOCK, -1)), pages[..., split:].unflatten(-1, (BLOCK, -1)), scale)
    return x.transpose(1, 2).flatten(2, 3)


def _attend_plain(s):
    hq, hk, d = s["hq"], s["hk"], s["d"]
    new = s["q_start"][1:] - s["q_start"][:-1]
    step = torch.arange(s["max_q"], device="cuda")
    at = s["q_start"][:-1, None] + step  # [B, Q]: row of each request's new tokens, padded to the longest
    live = step < new[:, None]
    q = s["q"].float()[at.clamp(max=s["q"].shape[0] - 1)].unflatten(-1, (hk, hq // hk, d))  # [B, Q, hk, G, D]
    q = q.permute(0, 2, 1, 3, 4).flatten(2, 3)  # [B, hk, Q * G, D]
    scores = torch.matmul(q, _gather(s["k_cache"], s["block_tables"], s["k_scale"], d).transpose(-1, -2)) * s["scale"]
    pos = (s["seq_lens"] - new)[:, None] + step
    key = torch.arange(scores.shape[-1], device="cuda")
    mask = (key <= pos[..., None]).repeat_interleave(hq // hk, 1)[:, None]  # [B, 1, Q * G, S]
    scores.masked_fill_(~mask, float("-inf"))
    p = torch.exp(scores.sub_(scores.amax(-1, keepdim=True)))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, _gather(s["v_cache"], s["block_tables"], s["v_scale"], d)) / total
    o = o.unflatten(2, (-1, hq // hk)).permute(0, 2, 1, 3, 4).flatten(2)  # [B, Q, hq * D]
    return o[live].bfloat16()


# ------------------------------------------------------------------------------------------------- 64 bits
def _exact_values(codes, scales, scale):
    sign = 1.0 - 2.0 * (codes >> 3).double()
    e, m = (codes >> 1 & 3).double(), (codes & 1).double()
    v = sign * torch.where(e == 0, m / 2, (1 + m / 2) * 2 ** (e - 1))
    return v * scales.double().repeat_interleave(16, -1) * scale


def _exact_rows(pages, d, scale):
    """fp64 rows [n * 64, D] of one head's pages [n, bytes]."""
    split = BLOCK * d // 2
    b = pages[:, :split].reshape(-1, d // 2)
    codes = torch.stack((b % 16, b // 16), -1).reshape(-1, d)
    scales = pages[:, split:].reshape(-1, d // 16).view(torch.float8_e4m3fn)
    return _exact_values(codes, scales.double(), scale)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "copy":
        return None  # no computed numbers
    hq, hk, d = case["hq"], case["hk"], case["d"]
    if case["op"] == "write":
        x = s["qkv"].double().view(case["tokens"], hq + 2 * hk, d)
        half = case["rot"] // 2
        cs = s["cos_sin"].double()[s["positions"]]
        z = torch.complex(x[..., :half], x[..., half:2 * half]) * torch.complex(cs[:, None, :half], cs[:, None, half:])
        y = torch.cat((z.real, z.imag, x[..., 2 * half:]), -1)
        grid = torch.arange(0x7F, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).double()

        def cached(rows, scale):
            rows = (rows / scale).unflatten(-1, (-1, 16))
            want = (rows.abs().amax(-1) / 6).clamp(2.0 ** -9, 448.0)
            up = torch.searchsorted(grid, want).clamp(1, 0x7E)
            lo, hi = grid[up - 1], grid[up]
            low = (want - lo < hi - want) | ((want - lo == hi - want) & (up % 2 == 1))
            sc = torch.where(low, lo, hi)[..., None]
            mag = torch.tensor(E2M1, dtype=torch.float64, device="cuda")
            r = rows.abs() / sc
            j = torch.searchsorted(mag, r).clamp(1, 7)
            down = (r - mag[j - 1] < mag[j] - r) | ((r - mag[j - 1] == mag[j] - r) & (j % 2 == 1))
            v = torch.where(down, mag[j - 1], mag[j]) * torch.sign(rows) * sc * scale
            return torch.where((s["slots"] >= 0)[:, None, None], v.flatten(-2), 0.0)

        return y[:, :hq].flatten(1), cached(y[:, hq:hq + hk], s["k_scale"]), cached(x[:, hq + hk:], s["v_scale"])
    out = torch.zeros(s["q"].shape[0], hq, d, dtype=torch.float64, device="cuda")
    g, row = hq // hk, 0
    for i, (new, n) in enumerate(_lengths(case)):
        used = s["block_tables"][i, : -(-n // BLOCK)].long()
        pos = torch.arange(n - new, n, device="cuda")
        for h in range(hk):
            k = _exact_rows(s["k_cache"][used, h], d, s["k_scale"])[:n]
            v = _exact_rows(s["v_cache"][used, h], d, s["v_scale"])[:n]
            for lo in range(0, new, 1024):  # rows of a bounded score matrix
                hi = min(new, lo + 1024)
                q = s["q"][row + lo:row + hi].view(hi - lo, hq, d)[:, h * g:(h + 1) * g].double()
                sc = torch.einsum("tgd,nd->tgn", q, k) * s["scale"]
                sc = torch.where(torch.arange(n, device="cuda") <= pos[lo:hi, None, None], sc, -math.inf)
                out[row + lo:row + hi, h * g:(h + 1) * g] = torch.softmax(sc, -1) @ v
        row += new
    return out.flatten(1)
