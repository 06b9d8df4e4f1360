"""Measured cases of the serving operators for many sequences at once: attention over packed
prompts, the paged 4-bit key/value cache that they fill, single-token attention over that cache, and
the moves of its pages.

Each case runs one pass of one of them, either through the framework's entry points (``own``) or in
a plain form of elementary torch operations in 32 bits.  Four kinds of case:

``packed``  causal attention of whole prompts of different lengths, packed row after row
``write``   rows of keys and values written into the pages of a 4-bit cache, and read back
``decode``  attention of one new token a sequence over its pages
``pages``   one scheduling step: sequences forked, finished ones freed, the pool compacted

The cache's format (the framework's documentation has it too).  Positions are held in pages of
``page`` positions; a page holds, for each layer apart, ``n_kv`` heads of ``page / 16`` blocks of 16
positions.  A block is ``18 * head_dim`` bytes: key codes, value codes, key scales, value scales.  32
consecutive values of a head share a scale d (16-bit float), and value = d * (code - 8).
"""
import math
import random
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _case(name, kind, dtype, heads, n_kv, hd, seqs, longest, ragged, **more):
    return dict(name=name, kind=kind, dtype=dtype, heads=heads, n_kv=n_kv, hd=hd, seqs=seqs, longest=longest,
                ragged=ragged, **more)


def listed():
    return [
        # a few short chat turns that arrive together at a small model: latency
        _case("packed_short_f16", "packed", "f16", 8, 2, 64, 5, 61, True),
        # prompts of a server tick on a model with as many key/value heads as query heads (the 7B's layer)
        _case("packed_mha_f16", "packed", "f16", 32, 32, 128, 6, 2048, True),
        # the same with grouped heads (the 70B's layer), to the longest prompt that it takes
        _case("packed_gqa_bf16", "packed", "bf16", 64, 8, 128, 8, 4096, True),
        # one long document
        _case("packed_long_bf16", "packed", "bf16", 64, 8, 128, 1, 16383, False),
        # the first tokens of one answer of a small model: latency
        _case("decode_first_f32", "decode", "f32", 4, 2, 64, 1, 33, False, page=16),
        # single-stream decode at the end of the 7B's context, with the 32-bit activations of the decode engine
        _case("decode_mha_f32", "decode", "f32", 32, 32, 128, 1, 2047, False, page=64),
        # a full batch of the 70B, each sequence somewhere in its context
        _case("decode_batch_f16", "decode", "f16", 64, 8, 128, 64, 4096, True, page=64),
        # a few very long contexts
        _case("decode_long_bf16", "decode", "bf16", 64, 8, 128, 8, 131072, True, page=64),
        # the new token of each sequence of a batch
        _case("write_token_f32", "write", "f32", 64, 8, 128, 64, 1, False, page=64),
        # the rows of the prompts of a server tick
        _case("write_prompts_f16", "write", "f16", 64, 8, 128, 16, 4096, True, page=64),
        # parallel sampling of a small model
        _case("pages_small", "pages", "f16", 8, 2, 64, 6, 300, True, page=16, layers=2, pool=192, forks=3, finished=2,
              moves=9),
        # a busy server of the 70B (all 80 layers): a beam is forked, finished answers go, the pool is compacted
        _case("pages_80_layers", "pages", "f16", 64, 8, 128, 48, 2048, True, page=64, layers=80, pool=1100, forks=24,
              finished=12, moves=230),
    ]


def _between(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["packed", "packed", "decode", "decode", "decode", "write", "pages"])
    n_kv, group = rng.choice([(1, 8), (2, 1), (2, 4), (2, 7), (4, 3), (8, 1), (8, 4), (8, 8), (32, 1), (4, 16)])
    hd = rng.choice([64, 128, 128, 128])
    c = dict(kind=kind, dtype=rng.choice(["f16", "bf16"]), heads=n_kv * group, n_kv=n_kv, hd=hd)
    if kind == "packed":
        c["seqs"] = _between(rng, 1, 40)
        # the plain form holds all scores of a pass at once: 32 bits for each of heads * seqs * longest^2
        most = int(math.sqrt(1.0e10 / (c["heads"] * c["seqs"])))
        c["longest"] = _between(rng, 3, min(8192, most))
        c["ragged"] = rng.random() < 0.8
        return c
    c["page"] = rng.choice([16, 32, 48, 64, 128])
    if kind == "pages":
        c["layers"] = _between(rng, 1, 32)
        c["seqs"] = rng.randint(4, 32)
        c["longest"] = _between(rng, 40, 1500)
        c["ragged"] = True
        c["forks"], c["finished"] = rng.randint(1, c["seqs"] // 2), rng.randint(1, c["seqs"] // 4)
        kept = sum(-(-n // c["page"]) for n in lengths(c)[c["finished"]:])
        gone = sum(-(-n // c["page"]) for n in lengths(c)[:c["finished"]])
        c["pool"] = kept + gone + c["forks"] + rng.randint(3, 90)
        c["moves"] = rng.randint(0, min(kept, c["pool"] - kept - c["forks"]) // 2)
        return c
    c["dtype"] = rng.choice(["f32", "f16", "bf16"])
    c["ragged"] = rng.random() < 0.8
    if kind == "decode":
        c["hd"] = rng.choice([64, 128, 128, 256])
        c["seqs"] = _between(rng, 1, 96)
        c["longest"] = _between(rng, 1, min(60000, int(6.0e8 / (c["seqs"] * n_kv * c["hd"]))))
    else:
        c["hd"] = rng.choice([64, 128, 256])
        c["seqs"] = _between(rng, 1, 64)
        c["longest"] = _between(rng, 1, min(4096, int(6.0e7 / (c["seqs"] * n_kv * c["hd"]))))
    return c


def lengths(case):
    """The sequences' lengths: the case's alone, so that the work does not depend on the seed.  Ragged: from one token to the
    longest, which is there; the sequences of a decode batch may include one that has nothing yet."""
    n, top = case["seqs"], case["longest"]
    if not case["ragged"]:
        return [top] * n
    r = random.Random("%s %d %d %d" % (case["kind"], n, top, case["heads"]))
    got = [r.randint(max(1, top // 8), top) for _ in range(n)]
    got[r.randrange(n)] = top
    if n >= 4:
        short = r.choice([i for i in range(n) if got[i] != top] or [0])
        got[short] = 0 if case["kind"] == "decode" else 1
    return got


def block_bytes(hd):
    return 18 * hd


def page_bytes(case):
    return case["n_kv"] * (case["page"] // 16) * block_bytes(case["hd"])


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    n, hd, heads, n_kv = lengths(case), case["hd"], case["heads"], case["n_kv"]
    total = sum(n)
    if case["kind"] == "packed":
        return {"bytes": total * hd * size * (2 * heads + 2 * n_kv), "flops": sum(4.0 * hd * heads * x * (x + 1) / 2 for x in n)}
    if case["kind"] == "decode":
        return {"bytes": total * n_kv * block_bytes(hd) / 16 + 2 * case["seqs"] * heads * hd * size, "flops": 4.0 * hd * heads * total}
    if case["kind"] == "write":  # rows read, codes written, codes read, rows written
        return {"bytes": total * n_kv * 2 * (2 * hd * size + block_bytes(hd) / 16), "flops": 0}
    parents = lengths(case)[case["finished"]:][:case["forks"]]
    copied = sum(x % case["page"] != 0 for x in parents) + case["moves"]
    return {"bytes": 2.0 * copied * case["layers"] * page_bytes(case) + 8 * case["pool"], "flops": 0}


# ---- the cache's format ----------------------------------------------------------------------------------------------


def unpack(blocks, hd):
    """(keys, values) in 32 bits, [..., 16 positions, hd], of blocks [..., 18 * hd] of bytes."""
    nb, at = hd // 32, 8 * hd
    lead = blocks.shape[:-1]
    shifts = torch.arange(0, 32, 4, device=blocks.device, dtype=torch.int32)
    k = blocks[..., :at].contiguous().view(torch.int32).view(*lead, 16, 4, nb, 1) >> shifts & 15
    k = k.transpose(-3, -2).reshape(*lead, 16, nb, 32)
    v = blocks[..., at:2 * at].contiguous().view(torch.int16).view(*lead, 4, 8, 2, 2, nb, 1).to(torch.int32) >> shifts[:4] & 15
    m = len(lead)
    v = v.permute(*range(m), m + 1, m + 3, m + 4, m, m + 2, m + 5).reshape(*lead, 16, nb, 32)
    d = blocks[..., 2 * at:].contiguous().view(torch.float16).view(*lead, 2, 16, nb, 1).float()
    return ((k - 8).float() * d[..., 0, :, :, :]).view(*lead, 16, hd), ((v - 8).float() * d[..., 1, :, :, :]).view(*lead, 16, hd)


def pack_codes(k, v, dk, dv):
    """The bytes of codes k, v [..., 16, hd] (whole numbers of 32 bits) and scales dk, dv [..., 16, hd / 32]."""
    lead, hd = k.shape[:-2], k.shape[-1]
    nb, m = hd // 32, k.dim() - 2
    shifts = torch.arange(0, 32, 4, device=k.device, dtype=torch.int32)
    k = (k.view(*lead, 16, nb, 4, 8) << shifts).sum(-1, dtype=torch.int32).transpose(-1, -2).contiguous()
    v = (v.view(*lead, 8, 2, nb, 4, 2, 4) << shifts[:4]).sum(-1, dtype=torch.int32).to(torch.int16)
    v = v.permute(*range(m), m + 3, m, m + 4, m + 1, m + 2).contiguous()
    d = torch.stack([dk, dv], -3).contiguous()
    parts = [x.reshape(*lead, -1).view(torch.uint8) for x in (k, v, d)]
    return torch.cat(parts, -1)


def quantise(x):
    """(codes, scales) of x [..., hd]: for 32 values d = m / -8 in 16 bits, m the value of the largest magnitude (the first of
    them), and code = round(value / d) + 8 in [0, 15]; a group with a value that is not finite has no number as its scale."""
    x = x.float().view(*x.shape[:-1], -1, 32)
    size = x.abs()
    lanes = torch.arange(32, device=x.device)
    first = torch.where(size == size.amax(-1, keepdim=True), lanes, 31).amin(-1, keepdim=True)
    d = (x.gather(-1, first) / -8).half()
    d = torch.where(torch.isfinite(x).all(-1, keepdim=True), d, float("nan"))
    wide = d.float()
    steps = torch.where(wide == 0, 0.0, x / wide)
    codes = (steps.round().nan_to_num(0) + 8).clamp(0, 15).int()
    return codes.flatten(-2), d.squeeze(-1)


# ---- inputs ----------------------------------------------------------------------------------------------------------


def _heads(gen, rows, heads, hd, spread=0.0):
    """Rows of head vectors: normal, and for keys a few channels of a much larger size, as trained projections have."""
    x = torch.randn(rows, heads, hd, device="cuda", generator=gen)
    if spread:
        x *= 1 + spread * (torch.rand(heads, hd, device="cuda", generator=gen) > 0.96)
    return x


def _tables(case, gen, used, width, seqs, pool):
    """Tables [seqs][width] with pages of the pool in an order of their own, each used once; -1 past a sequence's pages."""
    pages = torch.randperm(pool, device="cuda", generator=gen)[:sum(used)].int()
    counts = torch.tensor(used, device="cuda")
    at = torch.arange(width, device="cuda")
    ends = counts.cumsum(0)
    index = (ends - counts)[:, None] + at
    table = torch.where(at < counts[:, None], pages[index.clamp(max=max(0, len(pages) - 1))] if len(pages) else -1, -1)
    return table.int().contiguous()


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    kind, hd, n_kv, heads = case["kind"], case["hd"], case["n_kv"], case["heads"]
    dtype, n = DTYPES[case["dtype"]], lengths(case)
    lens = torch.tensor(n, dtype=torch.int32, device="cuda")
    cu = torch.cat([lens.new_zeros(1), lens.cumsum(0).int()])
    s = {"case": dict(case), "lens": lens, "cu": cu}
    if kind == "packed":
        s["q"] = _heads(gen, sum(n), heads, hd).to(dtype)
        s["k"] = _heads(gen, sum(n), n_kv, hd, 3.0).to(dtype)
        s["v"] = _heads(gen, sum(n), n_kv, hd).to(dtype)
        s["out"] = torch.empty_like(s["q"])
        return s
    page = case["page"]
    if kind == "pages":
        return _prepare_pages(s, case, gen, n)
    used = [-(-x // page) for x in n]
    width = max(1, max(used))
    s["pool_pages"] = pool = sum(used) + 3
    s["tables"] = _tables(case, gen, used, width, len(n), pool)
    s["pool"] = torch.empty(1, pool, n_kv, page // 16, block_bytes(hd), dtype=torch.uint8, device="cuda")
    if kind == "write":
        s["k"] = _heads(gen, sum(n), n_kv, hd, 3.0).to(dtype)
        s["v"] = _heads(gen, sum(n), n_kv, hd).to(dtype)
        s["start"] = torch.zeros_like(lens)
        s["pool"].zero_()
        s["k_back"], s["v_back"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
        return s
    # a cache that earlier steps filled: the codes of normal values are normal about 8, and scales vary by channel group
    flat = s["pool"].view(-1, block_bytes(hd))
    some = max(1, (1 << 28) // (16 * hd))
    for i in range(0, len(flat), some):
        m = min(some, len(flat) - i)
        codes = (torch.randn(2, m, 16, hd, device="cuda", generator=gen).mul_(2.6).round_().add_(8)).clamp_(0, 15).int()
        scales = torch.rand(2, m, 16, hd // 32, device="cuda", generator=gen).mul_(0.35).add_(0.2).half()
        scales *= torch.where(torch.rand(2, m, 16, hd // 32, device="cuda", generator=gen) < 0.5, -1, 1).half()
        flat[i:i + m] = pack_codes(codes[0], codes[1], scales[0], scales[1])
    s["q"] = _heads(gen, len(n), heads, hd).to(dtype)
    s["out"] = torch.empty_like(s["q"])
    return s


def _prepare_pages(s, case, gen, n):
    """A pool of which, once the first `finished` sequences are gone and the `forks` next ones have a copy each, exactly `moves`
    pages lie above the pages that are in use."""
    page, pool, finished, forks = case["page"], case["pool"], case["finished"], case["forks"]
    used = [-(-x // page) for x in n]
    kept, gone = sum(used[finished:]), sum(used[:finished])
    copies = sum(x % page != 0 for x in n[finished:][:forks])
    # The copies take the lowest free pages.  Those below the final count are taken first, so the lowest `copies` pages are free.
    live = kept + copies
    low = torch.randperm(live - copies, device="cuda", generator=gen) + copies
    high = torch.randperm(pool - live, device="cuda", generator=gen) + live
    moves = case["moves"]
    mine = torch.cat([low[:kept - moves], high[:moves]])
    mine = mine[torch.randperm(kept, device="cuda", generator=gen)]
    rest = torch.cat([low[kept - moves:], high[moves:]])
    rest = rest[torch.randperm(len(rest), device="cuda", generator=gen)][:gone]
    pages = torch.cat([rest, mine]).int()
    width, rows = max(used) + 1, len(n) + forks
    counts = torch.tensor(used, device="cuda")
    at = torch.arange(width, device="cuda")
    index = ((counts.cumsum(0) - counts)[:, None] + at).clamp(max=len(pages) - 1)
    meta = torch.zeros(rows * width + rows + pool, dtype=torch.int32, device="cuda")
    meta[:rows * width] = -1
    meta[:len(n) * width] = torch.where(at < counts[:, None], pages[index], -1).view(-1)
    meta[rows * width:rows * width + len(n)] = s["lens"]
    meta[rows * width + rows + pages.long()] = 1
    s.update(meta_before=meta, meta=meta.clone(), rows=rows, width=width)
    s["parents"] = torch.arange(finished, finished + forks, dtype=torch.int32, device="cuda")
    s["children"] = torch.arange(len(n), len(n) + forks, dtype=torch.int32, device="cuda")
    s["finished"] = torch.arange(finished, dtype=torch.int32, device="cuda")
    shape = (case["layers"], pool, case["n_kv"], page // 16, block_bytes(case["hd"]))
    size = math.prod(shape) // 4
    s["pool"] = torch.empty(size, dtype=torch.int32, device="cuda").random_(generator=gen).view(torch.uint8).view(shape)
    return s


def _split(s):
    """The parts of the state's numbers: tables [rows][width], lengths [rows], page counts [pool]."""
    r, w = s["rows"], s["width"]
    return s["meta"][:r * w].view(r, w), s["meta"][r * w:r * w + r], s["meta"][r * w + r:]


# ---- one pass --------------------------------------------------------------------------------------------------------


def run(s):
    return (_own if own else _plain)[s["case"]["kind"]](s)


def _plain_packed(s):
    n, top = s["lens"].long(), max(lengths(s["case"]))
    hd, n_kv, group = s["case"]["hd"], s["case"]["n_kv"], s["case"]["heads"] // s["case"]["n_kv"]
    at = torch.arange(top, device="cuda")
    here = at < n[:, None]  # [seqs][top]
    rows = (s["cu"][:-1].long()[:, None] + at).clamp(max=len(s["q"]) - 1)
    q = s["q"].float()[rows].view(len(n), top, n_kv, group, hd).permute(0, 2, 3, 1, 4).reshape(len(n), n_kv, group * top, hd)
    k = s["k"].float()[rows].permute(0, 2, 3, 1)
    v = torch.where(here[:, :, None, None], s["v"].float()[rows], 0).transpose(1, 2)
    p = torch.matmul(q * hd ** -0.5, k).view(len(n), n_kv, group, top, top)
    del q, k
    p.masked_fill_(~((at <= at[:, None]) & here[:, None, :])[:, None, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    p.div_(p.sum(-1, keepdim=True))
    o = torch.matmul(p.view(len(n), n_kv, group * top, top), v).view(len(n), n_kv, group, top, hd)
    return o.permute(0, 3, 1, 2, 4)[here].reshape(-1, n_kv * group, hd).to(s["q"].dtype)


def _positions(s):
    """For every row of the packed rows: its page and its place in the page."""
    n, cu, page = s["lens"].long(), s["cu"].long(), s["case"]["page"]
    total = s["k"].shape[0]
    seq = torch.repeat_interleave(torch.arange(len(n), device="cuda"), n, output_size=total)
    at = torch.arange(total, device="cuda") - cu[seq] + s["start"].long()[seq]
    return s["tables"].long()[seq, at // page], at % page


def _plain_write(s):
    hd, nb = s["case"]["hd"], s["case"]["hd"] // 32
    (ck, dk), (cv, dv) = quantise(s["k"]), quantise(s["v"])
    pages, at = _positions(s)
    blocks = s["pool"][0][pages, :, at // 16]  # the blocks of the rows, [rows][n_kv][bytes]: written row by row
    slot = at % 16
    shifts = torch.arange(0, 32, 4, device="cuda", dtype=torch.int32)
    lead = ck.shape[:2]
    wk = (ck.view(*lead, nb, 4, 8) << shifts).sum(-1, dtype=torch.int32).transpose(-1, -2).reshape(*lead, 4 * nb)
    wv = (cv.view(*lead, nb, 4, 2, 4) << shifts[:4]).sum(-1, dtype=torch.int32).to(torch.int16).permute(0, 1, 3, 4, 2)
    flat = s["pool"].view(-1)
    base = ((pages * lead[1])[:, None] + torch.arange(lead[1], device="cuda")) * (s["case"]["page"] // 16) + (at // 16)[:, None]
    base, slot = base * block_bytes(hd), slot[:, None]
    words, halves, scales = flat.view(torch.int32), flat.view(torch.int16), flat.view(torch.float16)
    words[(base + slot * (hd // 2))[..., None] // 4 + torch.arange(4 * nb, device="cuda")] = wk
    u, g, b = (torch.arange(m, device="cuda") for m in (4, 2, nb))
    place = (((u[:, None, None] * 8) * 2 + g[:, None]) * 2) * nb + b + ((slot // 2 * 4 + slot % 2) * nb)[..., None, None, None]
    halves[(base + 8 * hd)[..., None, None, None] // 2 + place] = wv
    scales[(base + 16 * hd)[..., None] // 2 + slot[..., None] * nb + b] = dk
    scales[(base + 17 * hd)[..., None] // 2 + slot[..., None] * nb + b] = dv
    blocks = s["pool"][0][pages, :, at // 16]
    k, v = unpack(blocks, hd)
    pick = slot[:, :, None, None].expand(-1, lead[1], 1, hd)
    return {"k": k.gather(2, pick)[:, :, 0].to(s["k"].dtype), "v": v.gather(2, pick)[:, :, 0].to(s["v"].dtype)}


def _plain_decode(s):
    hd, n_kv, heads = s["case"]["hd"], s["case"]["n_kv"], s["case"]["heads"]
    blocks = s["pool"][0][s["tables"].long().clamp(min=0)]  # [seqs][width][n_kv][page / 16][bytes]
    k, v = unpack(blocks.transpose(1, 2), hd)  # [seqs][n_kv][width][page / 16][16][hd]
    k, v = k.flatten(2, 4), v.flatten(2, 4)
    q = s["q"].float().view(-1, n_kv, heads // n_kv, hd)
    here = (torch.arange(k.shape[2], device="cuda") < s["lens"][:, None])[:, None, None]
    p = torch.where(here, torch.matmul(q * hd ** -0.5, k.transpose(-1, -2)), -math.inf)
    p = torch.where(here, (p - p.amax(-1, keepdim=True)).exp(), 0)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, 1)
    return o.view(-1, heads, hd).to(s["q"].dtype)


def _plain_pages(s):
    case, pool = s["case"], s["pool"].view(torch.int64)
    page = case["page"]
    s["meta"].copy_(s["meta_before"])
    tables, lens, refs = _split(s)
    parents, children, finished = s["parents"].long(), s["children"].long(), s["finished"].long()
    at = torch.arange(s["width"], device="cuda")
    every = torch.arange(case["pool"], device="cuda")

    # fork: whole pages are shared, a last page with room is copied into the lowest free page
    n = lens[parents]
    partial = n % page != 0
    source = tables[parents, (n // page).clamp(max=s["width"] - 1).long()].long()
    free = torch.where(refs == 0, every, case["pool"]).sort().values
    target = free[(partial.cumsum(0) - 1).clamp(min=0)]
    pool[:, target[partial]] = pool[:, source[partial]]
    whole = at < (n // page)[:, None]
    shared = tables[parents].long()
    tables[children] = torch.where(whole, shared, torch.where((at == (n // page)[:, None]) & partial[:, None], target[:, None], -1)).int()
    lens[children] = n
    refs.scatter_add_(0, shared.clamp(min=0).view(-1), whole.view(-1).int())
    refs.scatter_add_(0, target, partial.int())

    # free
    old = tables[finished].long()
    held = at < ((lens[finished] + page - 1) // page)[:, None]
    refs.scatter_add_(0, old.clamp(min=0).view(-1), -held.view(-1).int())
    tables[finished], lens[finished] = -1, 0

    # compact: the pages in use above their count move, in order, to the free ones below it
    used = refs > 0
    live = used.sum()
    source, target = (used & (every >= live)).nonzero().view(-1), (~used & (every < live)).nonzero().view(-1)
    pool[:, target] = pool[:, source]
    to = every.clone()
    to[source] = target
    refs[target], refs[source] = refs[source], 0
    tables.copy_(torch.where(tables >= 0, to[tables.long().clamp(min=0)].int(), -1))
    return {"tables": tables, "lens": lens, "refs": refs, "pool": s["pool"].view(torch.int32)}


_plain = {"packed": _plain_packed, "write": _plain_write, "decode": _plain_decode, "pages": _plain_pages}


def _framework():
    if "google-classic_b200" not in sys.path:
        sys.path.insert(0, "google-classic_b200")
    from holo_b200 import attention, kv4
    return attention, kv4


def _own_packed(s):
    if "op" not in s:
        s["op"] = _framework()[0].attention_packed
    return s["op"](s["q"], s["k"], s["v"], s["cu"], out=s["out"])


def _cache(s):
    """The cache object that a user's program keeps, over this state's pool and tables."""
    if "cache" not in s:
        c = s["case"]
        tables, lens, refs = _split(s) if c["kind"] == "pages" else (s["tables"], s["lens"], None)
        s["cache"] = _framework()[1].Kv4Cache(n_layers=c.get("layers", 1), n_kv_heads=c["n_kv"], head_dim=c["hd"],
                                              page_tokens=c["page"], pool=s["pool"], tables=tables, lens=lens, refs=refs)
    return s["cache"]


def _own_write(s):
    cache = _cache(s)
    cache.append(0, s["k"], s["v"], s["cu"], s["start"])
    k, v = cache.read(0, s["cu"], s["start"], s["k_back"], s["v_back"])
    return {"k": k, "v": v}


def _own_decode(s):
    return _cache(s).attention(0, s["q"], out=s["out"])


def _own_pages(s):
    cache = _cache(s)
    s["meta"].copy_(s["meta_before"])
    cache.fork(s["parents"], s["children"])
    cache.release(s["finished"])
    cache.compact()
    return {"tables": cache.tables, "lens": cache.lens, "refs": cache.refs, "pool": s["pool"].view(torch.int32)}


_own = {"packed": _own_packed, "write": _own_write, "decode": _own_decode, "pages": _own_pages}


# ---- from the definitions, in 64 bits --------------------------------------------------------------------------------


def _block_values(raw, hd, first, codes_at, scales_at):
    """Values [positions][hd] in 64 bits of blocks [m][18 * hd] of bytes, by the definition of each value's place."""
    nb = hd // 32
    pos, dim = torch.meshgrid(torch.arange(16, device="cuda"), torch.arange(hd, device="cuda"), indexing="ij")
    b, r = dim // 32, dim % 32
    if first:  # key: 4 words a group of 8 values, the words of a quarter together
        nibble = (pos * (hd // 2) + ((r // 8) * nb + b) * 4) * 2 + r % 8
    else:  # value: halfwords of 4 values, in the order quarter, pair of positions, half of the quarter, position, group
        w = r // 4
        nibble = (((((w // 2) * 8 + pos // 2) * 2 + w % 2) * 2 + pos % 2) * nb + b) * 4 + r % 4
    byte = raw[:, (codes_at + nibble // 2).view(-1)].view(-1, 16, hd).int()
    code = torch.where((nibble % 2).bool(), byte // 16, byte % 16)
    low, high = (raw[:, (scales_at + (pos * nb + b) * 2 + i).view(-1)].view(-1, 16, hd).int() for i in (0, 1))
    bits = high * 256 + low
    sign, power, part = 1 - 2 * (bits // 32768).double(), bits // 1024 % 32, (bits % 1024).double()
    d = torch.where(power == 0, part * 2.0 ** -24, (1024 + part) * torch.pow(2.0, power.double() - 25))
    return (sign * d * (code - 8)).view(-1, hd)


def _attend(q, k, v, causal):
    w = q.double() @ k.double().T / math.sqrt(q.shape[-1])
    if causal:
        rows = len(k) - len(q) + torch.arange(len(q), device="cuda")
        w = w.masked_fill(torch.arange(len(k), device="cuda") > rows[:, None], -math.inf)
    return torch.softmax(w, -1) @ v.double()


def exact(case, seed):
    s = prepare(case, seed)
    kind, n, hd = case["kind"], lengths(case), case["hd"]
    group = case["heads"] // case["n_kv"]
    if kind == "pages":
        return None  # whole numbers only
    if kind == "packed":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        a = 0
        for x in n:
            for h in range(case["heads"]):
                for i in range(0, x, 4096):
                    e = min(x, i + 4096)
                    out[a + i:a + e, h] = _attend(s["q"][a + i:a + e, h], s["k"][a:a + e, h // group], s["v"][a:a + e, h // group], True)
            a += x
        return out
    if kind == "write":
        back = {}
        for name in ("k", "v"):
            x = s[name].double().view(-1, 32)
            m = x.gather(1, (x.abs() >= x.abs().amax(1, keepdim=True)).int().argmax(1, keepdim=True))
            d = (m / -8).half().double()
            codes = torch.where(d == 0, 0.0, x / d).round().clamp(-8, 7)
            back[name] = (codes * d).view(s[name].shape)
        return back
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, x in enumerate(n):
        pages = s["tables"][i, :-(-x // case["page"])].long()
        for h in range(case["n_kv"] if x else 0):
            raw = s["pool"][0][pages, h].flatten(0, 1)
            k, v = (_block_values(raw, hd, first, c, d)[:x] for first, c, d in ((True, 0, 16 * hd), (False, 8 * hd, 17 * hd)))
            out[i, h * group:(h + 1) * group] = _attend(s["q"][i, h * group:(h + 1) * group], k, v, False)
    return out
