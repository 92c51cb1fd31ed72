"""The operators of a serving step over caches held in 4 bits: what a server calls around its decode.

Four kinds of call, each through a public entry point:

* ``attend`` - one decode step over paged 4-bit caches (``paged_attention.paged_attention_decode`` with packed pools
  and fp16 scales), also with several causal query tokens per sequence;
* ``append`` - new tokens' K/V quantised into those caches at their slots, and read back as rows
  (``kv_cache.kv4_append``, ``kv_cache.kv4_gather``), as a server that writes a prompt chunk and attends to it does;
* ``tables`` - the block tables and slot maps of a step from the requests' lengths (``kv_cache.release_blocks`` for
  the requests that ended, ``kv_cache.assign_slots`` for the others);
* ``rotary`` - q/k RMS norm, rotary positions of several axes and the cache write of a step
  (``kv_cache.qk_norm_mrope_append``).

The 4-bit caches. A row of ``dim`` values is cut into groups of ``group``; a group is held as 4-bit codes c with a
fp16 zero z and a fp16 scale s, and stands for c * s + z:

    lo, hi = the group's least and greatest value
    z = fp16(clamp(lo, +-65504)),  s = fp16(min((hi - lo) / 15, 65504)), in fp32, each operation rounded
    c = min(max(round((x - z) / s), 0), 15), ties to even; 0 where s is 0

Pools are uint8 ``[blocks, kv_heads, block, dim / 2]``, scales fp16 ``[blocks, kv_heads, groups, block, 2]`` (s, z).
Inside a page of one block and kv head (nibble 0 of a byte is the low one):

* K, row t: dword (dim/32) * a + j, nibble i holds dim 32 j + 8 a + i (a < 4, i < 8);
* V: rows 4 g .. 4 g + 3 share 2 dim bytes: byte (16-bit piece p = h + (dim/64) b of lane l at dword
  (dim/32) l + p; b picks rows 4 g + 2 b and + 1, low and high half), nibble 2 u + v of the half holds dim
  64 h + 32 u + 2 l + v.

Sizes are plain values; lengths come from ``len_draw``, so a case's work does not depend on the seed of its values.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
F16_MAX = 65504.0


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------


def _attend(name, batch, heads, kv_heads, dim, group, block, len_min, len_max, q_len=1, dtype="bf16", out="bf16",
            len_draw=1):
    return {"name": name, "kind": "attend", "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "group": group, "block": block, "len_min": len_min, "len_max": len_max, "q_len": q_len, "dtype": dtype,
            "out": out, "len_draw": len_draw}


def _append(name, tokens, kv_heads, dim, group, block, dtype="bf16", start=0, scattered=False):
    return {"name": name, "kind": "append", "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "group": group,
            "block": block, "dtype": dtype, "start": start, "scattered": scattered}


def _tables(name, batch, block, len_max, prompts, prompt_max, ended, width, len_draw=1):
    return {"name": name, "kind": "tables", "batch": batch, "block": block, "len_max": len_max, "prompts": prompts,
            "prompt_max": prompt_max, "ended": ended, "width": width, "len_draw": len_draw}


def _rotary(name, tokens, heads, kv_heads, dim, axes, block, dtype="bf16", proj="fp32", norm=True, interleaved=False):
    return {"name": name, "kind": "rotary", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "axes": axes, "block": block, "dtype": dtype, "proj": proj, "norm": norm, "interleaved": interleaved}


def listed():
    return [
        # the smallest decode: two short sequences of one kv head, bound by latency, launches and the call itself
        _attend("attend_small", 2, 16, 1, 128, 64, 128, 512, 512),
        # the flagship's decode step: 32 query and 8 kv heads, 32 sequences
        _attend("attend_serving", 32, 32, 8, 128, 64, 128, 1024, 8192),
        # the largest: few sequences with long contexts, whole rows as groups
        _attend("attend_long", 8, 64, 8, 128, 128, 128, 32768, 32768),
        # speculative verify, 8 causal query tokens, fine groups, pages of 32, fp16, an odd batch
        _attend("attend_verify", 13, 32, 8, 128, 32, 32, 700, 9000, q_len=8, dtype="fp16", out="fp16"),
        # small heads in pages of 16, fp32 output for a caller that merges further
        _attend("attend_d64_fp32", 37, 28, 4, 64, 32, 16, 300, 5000, out="fp32"),
        # the decode step's cache write: one token per sequence, anywhere in the pool
        _append("append_step", 32, 8, 128, 64, 128, scattered=True),
        # a prompt's cache write, of odd length and from the middle of a block on
        _append("append_prompt", 16001, 8, 128, 64, 128, start=37),
        # a chunk of a prompt of a fp16 model with small heads and pages of 16
        _append("append_chunk_fp16", 777, 4, 64, 32, 16, dtype="fp16", start=3),
        # a decode step's tables: one token for every request, a few that ended
        _tables("tables_decode", 256, 16, 8192, 0, 0, 5, 640),
        # a step that admits prompts among decodes
        _tables("tables_prompts", 1024, 32, 6000, 60, 8000, 40, 512),
        # the flagship's decode step of text and image positions
        _rotary("rotary_step", 32, 32, 8, 128, "16,24,24", 128),
        # a prompt with images or video: 16-bit projections, no norms
        _rotary("rotary_prompt", 9001, 32, 8, 128, "24,20,20", 64, proj="bf16", norm=False, interleaved=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: batches of 1 to 256 and lengths of 1 to 32768 of up to 1M (token, kv head) pairs, prompts of 1 to
    32768 tokens, 2 to 2048 requests, every block size, head size, group and type."""
    kind = rng.choice(["attend"] * 5 + ["append"] * 3 + ["tables"] * 2 + ["rotary"] * 2)
    block = rng.choice([16, 32, 64, 128])
    if kind == "attend":
        kv_heads, batch, q_len = rng.choice([1, 2, 4, 8]), _log(rng, 1, 256), rng.choice([1, 1, 1, 2, 4, 8])
        dim = rng.choice([64, 128, 128, 128, 256])
        dtype = rng.choice(["bf16", "bf16", "fp16"])
        heads = kv_heads * rng.choice([1, 2, 4, 5, 7, 8, 16])
        most = max(16, min(32768, int(1.3e8 / (batch * kv_heads * dim)), int(1.2e10 / (batch * q_len * heads * 4 * dim))))
        len_max = max(q_len, _log(rng, 1, most))
        c = _attend("", batch, heads, kv_heads, dim,
                    rng.choice([g for g in (32, 64, 128) if g <= dim <= 4 * g]), block,
                    max(q_len, int(len_max * rng.uniform(0.05, 1.0))), len_max, q_len, dtype,
                    rng.choice([dtype, dtype, "fp32"]), rng.randrange(1 << 20))
    elif kind == "append":
        dim = rng.choice([64, 128, 128, 256])
        kv_heads = rng.choice([1, 2, 4, 8])
        tokens = min(_log(rng, 1, 32768), int(2.5e8 / (12 * kv_heads * dim)))
        c = _append("", tokens, kv_heads, dim, rng.choice([g for g in (32, 64, 128) if g <= dim <= 4 * g]),
                    block, rng.choice(["bf16", "bf16", "fp16"]), rng.randrange(block), tokens <= 512 and rng.random() < 0.5)
    elif kind == "tables":
        batch = _log(rng, 2, 2048)
        prompts = rng.choice([0, rng.randint(0, max(1, batch // 8))])
        len_max, prompt_max = _log(rng, 1, 16000), _log(rng, 1, 4000)
        c = _tables("", batch, block, len_max, prompts, prompt_max, rng.randint(0, batch // 4),
                    (max(len_max, prompt_max) + block) // block + rng.randint(1, 9), rng.randrange(1 << 20))
    else:
        dim = rng.choice([64, 128, 128, 256])
        half, n = dim // 2, rng.choice([1, 2, 3, 3, 3, 4])
        interleaved = rng.random() < 0.4
        each = half // n  # interleaved: at most half / n pairs for each further axis
        rest = [rng.randint(max(1, each // 2), each if interleaved else each + each // 4) for _ in range(n - 1)]
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 4, 5, 7, 8])
        tokens = min(_log(rng, 1, 16384), int(2.2e8 / ((heads + 2 * kv_heads) * dim * 6)))
        c = _rotary("", tokens, heads, kv_heads, dim, ",".join(map(str, [half - sum(rest), *rest])), block,
                    rng.choice(["bf16", "bf16", "fp16"]), rng.choice(["fp32", "bf16", "fp16"]), rng.random() < 0.7,
                    interleaved)
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# The 4-bit format, in torch
# ---------------------------------------------------------------------------


def _quantised(x, group):
    """x [..., dim] of 16 bits -> codes [..., dim] (uint8), s and z [..., dim / group] (fp16)."""
    x = x.unflatten(-1, (-1, group))
    lo, hi = x.amin(-1).float(), x.amax(-1).float()
    z = lo.clamp(-F16_MAX, F16_MAX).half()
    s = ((hi - lo) / 15.0).clamp(max=F16_MAX).half()
    s64 = s.double().unsqueeze(-1)
    c = ((x.double() - z.double().unsqueeze(-1)) / torch.where(s64 > 0, s64, 1.0)).round().clamp(0, 15)
    return torch.where(s64 > 0, c, 0.0).to(torch.uint8).flatten(-2), s, z


def _values(codes, s, z, group):
    """fp32 values of codes [..., dim] with s and z [..., dim / group]."""
    c = codes.unflatten(-1, (-1, group)).float()
    return (c * s.float().unsqueeze(-1) + z.float().unsqueeze(-1)).flatten(-2)


def _k_view(pool):
    """[blocks, kv_heads, block, 4 a, dim/32 j, 4 bytes] of a K pool."""
    return pool.unflatten(-1, (4, -1, 4))


def _v_view(pool):
    """[blocks, kv_heads, block / 4 g, 2 b, 2 half, dim/64 h, 2 u, 16 l] of a V pool: a byte holds v = 0 (low) and 1."""
    n, hkv, block, row = pool.shape
    return pool.view(n, hkv, block // 4, 16, 2, row // 32, 2, 2).permute(0, 1, 2, 4, 6, 5, 7, 3)


def _k_bytes(codes):
    """codes [..., dim] -> [..., 4 a, dim/32 j, 4 bytes]."""
    c = codes.unflatten(-1, (-1, 4, 4, 2)).transpose(-4, -3)
    return c[..., 0] | (c[..., 1] << 4)


def _v_bytes(codes):
    """codes [..., dim] -> [..., dim/64 h, 2 u, 16 l]."""
    c = codes.unflatten(-1, (-1, 2, 16, 2))
    return c[..., 0] | (c[..., 1] << 4)


def _k_codes(b):
    c = torch.stack([b & 15, b >> 4], -1).flatten(-2)  # [..., a, j, 8 nibbles]
    return c.transpose(-3, -2).flatten(-3)


def _v_codes(b):
    return torch.stack([b & 15, b >> 4], -1).flatten(-4)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _randn(shape, gen, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _lengths(c):
    r = random.Random(c["len_draw"])
    return [r.randint(c["len_min"], c["len_max"]) for _ in range(c["batch"])]


def _pools(blocks, c):
    """Empty K and V pools and their scales."""
    page = (blocks, c["kv_heads"], c["block"], c["dim"] // 2)
    scales = (blocks, c["kv_heads"], c["dim"] // c["group"], c["block"], 2)
    return {"k": torch.zeros(page, dtype=torch.uint8, device="cuda"),
            "v": torch.zeros(page, dtype=torch.uint8, device="cuda"),
            "k_scale": torch.zeros(scales, dtype=torch.float16, device="cuda"),
            "v_scale": torch.zeros(scales, dtype=torch.float16, device="cuda")}


def _prepare_attend(c, gen):
    lens, block = _lengths(c), c["block"]
    per = [(n + block - 1) // block for n in lens]
    blocks = sum(per)
    s = _pools(blocks, c)
    # keys have channels of their own level, as projected keys do; values do not
    level = _randn((c["kv_heads"], 1, c["dim"]), gen)
    part = max(1, (1 << 26) // (c["kv_heads"] * block * c["dim"]))
    for at in range(0, blocks, part):
        shape = (min(part, blocks - at), c["kv_heads"], block, c["dim"])
        for name, x in (("k", _randn(shape, gen) + level), ("v", _randn(shape, gen))):
            codes, sc, z = _quantised(x.to(torch.bfloat16), c["group"])
            s[name + "_scale"][at:at + part] = torch.stack([sc, z], -1).transpose(2, 3)
            if name == "k":
                _k_view(s["k"])[at:at + part] = _k_bytes(codes)
            else:
                _v_view(s["v"])[at:at + part] = _v_bytes(codes).unflatten(2, (-1, 2, 2))
    # a table whose sequences take blocks all over the pool, as a server's do after a while
    perm = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros((c["batch"], max(per)), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = perm[at:at + n]
        at += n
    rows = (c["batch"], c["q_len"], c["heads"]) if c["q_len"] > 1 else (c["batch"], c["heads"])
    s |= {"q": _randn((*rows, c["dim"]), gen, DTYPES[c["dtype"]]), "table": table,
          "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "scale": 1.0 / math.sqrt(c["dim"]),
          "causal": c["q_len"] > 1, "out": torch.empty((*rows, c["dim"]), dtype=DTYPES[c["out"]], device="cuda")}
    return s


def _prepare_append(c, gen):
    block, tokens = c["block"], c["tokens"]
    blocks = (c["start"] + tokens + block - 1) // block + 3
    if c["scattered"]:  # one token each for many sequences
        slots = torch.randperm(blocks * block, generator=gen, device="cuda")[:tokens]
        if tokens > 8:
            slots[tokens // 3] = -1  # an idle sequence
    else:  # positions in order, their blocks anywhere in the pool
        order = torch.randperm(blocks, generator=gen, device="cuda")
        pos = c["start"] + torch.arange(tokens, device="cuda")
        slots = order[pos // block] * block + pos % block
    qkv = _randn((tokens, 4, c["kv_heads"], c["dim"]), gen, DTYPES[c["dtype"]])  # a projection's output: two parts are q
    return {**_pools(blocks, c), "key": qkv[:, 2], "value": qkv[:, 3], "slots": slots.to(torch.int32)}


def _requests(c):
    """Cached and new tokens of each request, and which have ended."""
    r = random.Random(c["len_draw"])
    order = list(range(c["batch"]))
    r.shuffle(order)
    prompts, ended = set(order[:c["prompts"]]), set(order[c["prompts"]:c["prompts"] + c["ended"]])
    lens = [0 if b in prompts else r.randint(1, c["len_max"]) for b in range(c["batch"])]
    new = [0 if b in ended else r.randint(1, c["prompt_max"]) if b in prompts else 1 for b in range(c["batch"])]
    return lens, new, ended


def _prepare_tables(c, gen):
    lens, new, ended = _requests(c)
    block = c["block"]
    per = [(n + block - 1) // block for n in lens]
    need = sum((n + m + block - 1) // block - p for n, m, p in zip(lens, new, per))
    pool = sum(per) + max(16, need + c["batch"] // 8 - sum(per[b] for b in ended) // 2)
    perm = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((c["batch"], c["width"]), -1, dtype=torch.int32, device="cuda")
    used = torch.tensor(per, device="cuda")[:, None] > torch.arange(c["width"], device="cuda")[None]
    table[used] = perm[:sum(per)]
    free = torch.full((pool,), -1, dtype=torch.int32, device="cuda")
    free[:pool - sum(per)] = perm[sum(per):]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return {"lens": i32(lens), "new": i32(new), "ended": i32([b in ended for b in range(c["batch"])]), "table": table,
            "free": free, "free_count": i32([pool - sum(per)]), "block": block, "tokens": sum(new) + sum(new) % 7}


def _prepare_rotary(c, gen):
    tokens, heads, hkv, dim, block = c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["block"]
    sections = [int(n) for n in c["axes"].split(",")]
    qkv = _randn((tokens, (heads + 2 * hkv) * dim), gen, DTYPES[c["proj"]])
    q, k, v = qkv.split([heads * dim, hkv * dim, hkv * dim], 1)
    # text, then an image of rows and columns: the axes' positions agree in the text
    at = torch.arange(tokens, device="cuda")
    side = max(1, int(math.sqrt(tokens / 2)))
    picture = at - tokens // 2
    pos = [at]
    for a in range(1, len(sections)):
        grid = picture // side if a % 2 else picture % side
        pos.append(torch.where(picture > 0, tokens // 2 + grid, at))
    if tokens <= 256:  # a decode step: every token at a place of its own
        pos = [p + torch.randint(0, 4096, (tokens,), generator=gen, device="cuda") for p in pos]
    most = tokens + 4096
    freq = 1.0 / (1.0e6 ** (torch.arange(dim // 2, device="cuda").double() / (dim // 2)))
    angle = torch.arange(most, device="cuda").double()[:, None] * freq
    blocks = (tokens + block - 1) // block
    cache = (blocks, block, hkv, dim)
    order = torch.randperm(blocks, generator=gen, device="cuda")
    s = {"q": q, "k": k, "v": v, "positions": torch.stack(pos).to(torch.int32).contiguous(), "sections": sections,
         "cos": torch.cat([angle.cos()] * 2, 1).float(), "sin": torch.cat([angle.sin()] * 2, 1).float(),
         "slots": (order[at // block] * block + at % block).to(torch.int32), "heads": heads,
         "k_cache": torch.zeros(cache, dtype=DTYPES[c["dtype"]], device="cuda"),
         "v_cache": torch.zeros(cache, dtype=DTYPES[c["dtype"]], device="cuda"), "interleaved": c["interleaved"],
         "inv_rms": None, "q_w": None, "k_w": None}
    if c["norm"]:
        s["inv_rms"] = 0.5 + torch.rand(tokens, generator=gen, device="cuda")
        s["q_w"], s["k_w"] = 1 + 0.1 * _randn((dim,), gen), 1 + 0.1 * _randn((dim,), gen)
    return s


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    made = {"attend": _prepare_attend, "append": _prepare_append, "tables": _prepare_tables,
            "rotary": _prepare_rotary}[case["kind"]](case, gen)
    return {"kind": case["kind"], "group": case.get("group"), **made}


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def _attend_own(s):
    from simpler_amd import paged_attention as pa

    return pa.paged_attention_decode(s["q"], s["k"], s["v"], s["table"], s["lens"], s["out"], s["scale"],
                                     causal=s["causal"], k_scale=s["k_scale"], v_scale=s["v_scale"])


def _attend_plain(s):
    table, q = s["table"].long(), s["q"].float()
    batch, heads, dim = q.shape[0], q.shape[-2], q.shape[-1]
    block, hkv = s["k"].shape[2], s["k"].shape[1]
    q_len, group = (q.shape[1] if q.dim() == 4 else 1), heads // hkv
    kc, vc = _k_codes(_k_view(s["k"])[table]), _v_codes(_v_view(s["v"])[table])
    vc = vc.flatten(3, 5)
    ks, vs = s["k_scale"][table].transpose(3, 4), s["v_scale"][table].transpose(3, 4)
    k, v = (_values(c, x[..., 0], x[..., 1], s["group"]).transpose(1, 2).flatten(2, 3)
            for c, x in ((kc, ks), (vc, vs)))  # [batch, kv head, token, dim]
    q = q.view(batch, q_len, hkv, group, dim).transpose(1, 2).reshape(batch, hkv, q_len * group, dim)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * s["scale"]
    seen = s["lens"][:, None] - (q_len - 1) + torch.arange(q_len, device="cuda").repeat_interleave(group)
    if not s["causal"]:
        seen = s["lens"][:, None].expand_as(seen)
    x = x.masked_fill(torch.arange(k.shape[2], device="cuda") >= seen[:, None, :, None], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-1e30))
    o = torch.matmul(p / p.sum(-1, keepdim=True).clamp_min(1e-30), v)
    o = o.view(batch, hkv, q_len, group, dim).transpose(1, 2)
    return o.reshape(s["out"].shape).to(s["out"].dtype)


def _append_own(s):
    from simpler_amd import kv_cache

    kv_cache.kv4_append(s["key"], s["value"], s["slots"], s["k"], s["v"], s["k_scale"], s["v_scale"])
    key, value = kv_cache.kv4_gather(s["slots"], s["k"], s["v"], s["k_scale"], s["v_scale"], dtype=s["key"].dtype)
    return {"key": key, "value": value, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _append_plain(s):
    block = s["k"].shape[2]
    there = s["slots"] >= 0
    slot = s["slots"].long()[there]
    blk, off = slot // block, slot % block
    got = {"k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    codes, sc, z = _quantised(s["key"][there], s["group"])
    _k_view(s["k"])[blk, :, off] = _k_bytes(codes)
    s["k_scale"][blk, :, :, off] = torch.stack([sc, z], -1)
    codes, sc, z = _quantised(s["value"][there], s["group"])
    _v_view(s["v"])[blk, :, off // 4, off % 4 // 2, off % 2] = _v_bytes(codes)
    s["v_scale"][blk, :, :, off] = torch.stack([sc, z], -1)
    kb, vb = _k_view(s["k"])[blk, :, off], _v_view(s["v"])[blk, :, off // 4, off % 4 // 2, off % 2]
    ks, vs = s["k_scale"][blk, :, :, off], s["v_scale"][blk, :, :, off]
    for name, c, x in (("key", _k_codes(kb), ks), ("value", _v_codes(vb), vs)):
        got[name] = torch.zeros(s[name].shape, dtype=s[name].dtype, device="cuda")
        got[name][there] = _values(c, x[..., 0], x[..., 1], s["group"]).to(s[name].dtype)
    return got


def _tables_own(s):
    from simpler_amd import kv_cache

    freed = kv_cache.release_blocks(s["ended"], s["lens"], s["table"], s["free"], s["free_count"], s["block"])
    step = kv_cache.assign_slots(s["new"], freed.context_lens, s["table"], s["free"], freed.free_count, s["block"],
                                 s["tokens"])
    return {"slots": step.slot_mapping, "positions": step.positions, "requests": step.requests, "starts": step.starts,
            "lens": step.context_lens, "granted": step.granted, "free_count": step.free_count, "table": s["table"],
            "free": s["free"]}


def _tables_plain(s):
    block, width, tokens = s["block"], s["table"].shape[1], s["tokens"]
    lens, table, free = s["lens"].long(), s["table"], s["free"]
    col, batch = torch.arange(width, device="cuda"), lens.shape[0]
    # the ended requests' blocks go on top of the free list, request by request
    per = torch.where(s["ended"] != 0, (lens + block - 1) // block, 0)
    first = s["free_count"].long() + per.cumsum(0) - per
    gone = col < per[:, None]
    free[(first[:, None] + col)[gone]] = table[gone]
    count = s["free_count"].long() + per.sum()
    lens = torch.where(s["ended"] != 0, 0, lens)
    # the others take theirs from its top, request by request, each all or nothing
    new = s["new"].long()
    ends = new.cumsum(0)
    fits = (lens + new <= width * block) & (ends <= tokens)
    had = (lens + block - 1) // block
    need = torch.where(fits, (lens + new + block - 1) // block - had, 0)
    upto = need.cumsum(0)
    fits &= (need == 0) | (upto <= count)
    at = col - had[:, None]
    taken = (at >= 0) & (at < need[:, None]) & fits[:, None]
    table[taken] = free[(count - 1 - (upto - need)[:, None] - at)[taken]]
    left = count - torch.where(fits, need, 0).sum()
    granted = torch.where(fits, new, 0)
    # every new token's request, position and slot; -1 past the last one and where the request got nothing
    t = torch.arange(tokens, device="cuda")
    req = torch.searchsorted(ends, t, right=True).clamp(max=batch - 1)
    pos = lens[req] + t - (ends - new)[req]
    ok = (t < ends[-1]) & fits[req]
    phys = table[req, (pos // block).clamp(max=width - 1)].long()
    i32 = torch.int32
    return {"slots": torch.where(ok, phys * block + pos % block, -1).to(i32),
            "positions": torch.where(ok, pos, -1).to(i32), "requests": torch.where(ok, req, -1).to(i32),
            "starts": torch.cat([ends.new_zeros(1), ends]).to(i32), "lens": (lens + granted).to(i32),
            "granted": granted.to(i32), "free_count": left.reshape(1).to(i32), "table": table, "free": free}


def _rotary_own(s):
    from simpler_amd import kv_cache

    q = kv_cache.qk_norm_mrope_append(s["q"], s["k"], s["v"], s["positions"], s["sections"], s["cos"], s["sin"],
                                      s["slots"], s["k_cache"], s["v_cache"], s["heads"], interleaved=s["interleaved"],
                                      inv_rms=s["inv_rms"], q_norm_weight=s["q_w"], k_norm_weight=s["k_w"], eps=EPS)
    return {"q": q, "k": s["k_cache"], "v": s["v_cache"]}


def _axis_of_pair(sections, interleaved):
    """The axis that turns each pair of dims."""
    n, half = len(sections), sum(sections)
    pair = torch.arange(half, device="cuda")
    if interleaved:
        size = torch.tensor(sections, device="cuda")
        return torch.where(pair < n * size[pair % n], pair % n, 0)
    return torch.repeat_interleave(torch.arange(n, device="cuda"), torch.tensor(sections, device="cuda"))


def _rotary_plain(s):
    tokens, dim = s["q"].shape[0], s["cos"].shape[1]
    half = dim // 2
    row = s["positions"].long()[_axis_of_pair(s["sections"], s["interleaved"])].t()  # [tokens, pair]
    pair = torch.arange(half, device="cuda")
    cos = torch.cat([s["cos"][row, pair], s["cos"][row, pair + half]], 1)[:, None]
    sin = torch.cat([s["sin"][row, pair], s["sin"][row, pair + half]], 1)[:, None]
    inv = 1.0 if s["inv_rms"] is None else s["inv_rms"][:, None, None]

    def turned(x, w):
        x = x.float().view(tokens, -1, dim) * inv
        if w is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        return x * cos + torch.cat([-x[..., half:], x[..., :half]], -1) * sin

    dtype, block = s["k_cache"].dtype, s["k_cache"].shape[1]
    slot = s["slots"].long()
    s["k_cache"][slot // block, slot % block] = turned(s["k"], s["k_w"]).to(dtype)
    s["v_cache"][slot // block, slot % block] = (s["v"].float().view(tokens, -1, dim) * inv).to(dtype)
    return {"q": turned(s["q"], s["q_w"]).to(dtype), "k": s["k_cache"], "v": s["v_cache"]}


def run(state):
    kind = state["kind"]
    if own:
        return {"attend": _attend_own, "append": _append_own, "tables": _tables_own, "rotary": _rotary_own}[kind](state)
    return {"attend": _attend_plain, "append": _append_plain, "tables": _tables_plain, "rotary": _rotary_plain}[kind](state)


def work(case):
    c = case
    if c["kind"] == "attend":
        lens = _lengths(c)
        row = c["dim"] // 2 + 4 * (c["dim"] // c["group"])
        rows = c["batch"] * c["q_len"] * c["heads"]
        blocks = sum((n + c["block"] - 1) // c["block"] for n in lens)
        pairs = sum(c["q_len"] * n - (c["q_len"] * (c["q_len"] - 1) // 2 if c["q_len"] > 1 else 0) for n in lens)
        return {"bytes": sum(lens) * c["kv_heads"] * 2 * row + rows * c["dim"] * (2 + DTYPES[c["out"]].itemsize) +
                4 * (blocks + c["batch"]), "flops": pairs * c["heads"] * 4 * c["dim"]}
    if c["kind"] == "append":  # 16-bit rows in and out, their 4-bit form written and read
        row = 2 * c["dim"] + c["dim"] // 2 + 4 * (c["dim"] // c["group"])
        return {"bytes": 2 * c["tokens"] * (2 * c["kv_heads"] * row + 4), "flops": 0}
    if c["kind"] == "tables":
        lens, new, ended = _requests(c)
        b = c["block"]
        moved = sum((lens[r] + b - 1) // b for r in ended)
        moved += sum((n + m + b - 1) // b - (n + b - 1) // b for n, m in zip(lens, new))
        return {"bytes": 4 * (7 * c["batch"] + 2 * moved + 3 * (sum(new) + sum(new) % 7)), "flops": 0}
    values = c["tokens"] * (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
    axes = len(c["axes"].split(","))
    return {"bytes": values * (DTYPES[c["proj"]].itemsize + 2) + c["tokens"] * (4 * axes + 4 + 8 * c["dim"]),
            "flops": 0}


# ---------------------------------------------------------------------------
# The definitions, in 64 bits
# ---------------------------------------------------------------------------


def _exact_pages(pool, scales, ids, is_k, group):
    """fp64 rows [kv heads, tokens, dim] of the pages `ids`, nibble by nibble from the format's description."""
    pages, sc = pool[ids], scales[ids].double()
    n, hkv, block, row = pages.shape
    dim = 2 * row
    flat = pages.reshape(n, hkv, -1)
    t = torch.arange(block, device=pool.device)[:, None]
    d = torch.arange(dim, device=pool.device)[None, :]
    if is_k:
        a, j, i = d % 32 // 8, d // 32, d % 8
        nibble = t * dim + 8 * ((dim // 32) * a + j) + i
    else:
        h, u, lane, v = d // 64, d % 64 // 32, d % 32 // 2, d % 2
        dword = (t // 4) * (dim // 2) + (dim // 32) * lane + (dim // 64) * (t % 4 // 2) + h
        nibble = 8 * dword + 4 * (t % 2) + 2 * u + v
    byte = flat[:, :, (nibble // 2).flatten()].reshape(n, hkv, block, dim)
    code = torch.where(nibble % 2 == 1, byte >> 4, byte & 15).double()
    g = (d // group).expand(block, dim)
    s, z = (sc[:, :, g, t.expand(block, dim), w] for w in (0, 1))
    return (code * s + z).transpose(0, 1).reshape(hkv, n * block, dim)


def _exact_attend(c, s):
    q_len, hkv, dim = c["q_len"], c["kv_heads"], c["dim"]
    group = c["heads"] // hkv
    q_all = s["q"].double().view(c["batch"], q_len, hkv, group, dim)
    out = torch.empty((c["batch"], q_len, c["heads"], dim), dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"].tolist()):
        ids = s["table"][b, :(n + c["block"] - 1) // c["block"]].long()
        k = _exact_pages(s["k"], s["k_scale"], ids, True, c["group"])[:, :n]
        v = _exact_pages(s["v"], s["v_scale"], ids, False, c["group"])[:, :n]
        for i in range(q_len):
            m = n - (q_len - 1 - i) if s["causal"] else n
            x = (q_all[b, i][:, :, None, :] * k[:, None, :m]).sum(-1) if m * c["heads"] * dim < 1 << 24 else \
                torch.matmul(q_all[b, i], k[:, :m].transpose(1, 2).contiguous())
            p = torch.softmax(x * s["scale"], -1)
            out[b, i] = torch.matmul(p, v[:, :m].contiguous()).reshape(c["heads"], dim)
    return out.view(s["out"].shape)


def _exact_append(c, s):
    got = {"k_scale": None, "v_scale": None}
    idle = s["slots"] < 0
    for name in ("key", "value"):
        x = s[name].reshape(c["tokens"], c["kv_heads"], -1, c["group"])
        lo, hi = x.min(-1, keepdim=True).values.float(), x.max(-1, keepdim=True).values.float()
        zero = lo.clip(-F16_MAX, F16_MAX).half().double()
        step = ((hi - lo) / 15.0).clip(max=F16_MAX).half().double()
        code = torch.where(step > 0, torch.round((x.double() - zero) / step.clip(min=2.0 ** -30)), 0.0).clip(0, 15)
        got[name] = (code * step + zero).reshape(s[name].shape)
        got[name][idle] = 0.0
    return got


def _exact_rotary(c, s):
    half, n = c["dim"] // 2, len(s["sections"])
    axis = []
    for i in range(half):
        if c["interleaved"]:
            axis.append(i % n if i < n * s["sections"][i % n] else 0)
        else:
            axis.append(next(a for a in range(n) if i < sum(s["sections"][:a + 1])))
    got = {"k": s["k_cache"].double(), "v": s["v_cache"].double()}
    cos, sin = (torch.stack([t[s["positions"][a].long(), i] for i, a in enumerate(axis)], 1).double()[:, None, :]
                for t in (s["cos"], s["sin"]))
    inv = 1.0 if s["inv_rms"] is None else s["inv_rms"].double()[:, None, None]

    def complex_turn(x, w):
        x = x.double().reshape(c["tokens"], -1, c["dim"]) * inv
        if w is not None:
            x = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * w.double()
        z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * torch.complex(cos, sin)
        return torch.cat([z.real, z.imag], -1)

    slot = s["slots"].long()
    got["k"].view(-1, c["kv_heads"], c["dim"])[slot] = complex_turn(s["k"], s["k_w"])
    got["v"].view(-1, c["kv_heads"], c["dim"])[slot] = s["v"].double().reshape(c["tokens"], -1, c["dim"]) * inv
    got["q"] = complex_turn(s["q"], s["q_w"])
    return got


def exact(case, seed):
    if case["kind"] == "tables":
        return None
    s = prepare(case, seed)
    return {"attend": _exact_attend, "append": _exact_append, "rotary": _exact_rotary}[case["kind"]](case, s)
