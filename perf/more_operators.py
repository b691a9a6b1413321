"""A paged cache held in 8 or 4 bits a value, as measurable cases.

Three operators: the rotary write of new tokens into such a cache (with the
read of what it then holds for them), the read of whole sequences back into
ordinary rows, and attention of a batch of sequences' new tokens over the cache.
Each listed case stands for a use named at its entry; draw() gives more of the
same ranges.

The format. Of each head's row, 32 neighbouring elements share a power of two
2^(E - 127), one byte E; each is a code in e4m3 (8 bits) or e2m1 (4 bits, two to
a byte, the even element in the low half) and stands for 2^(E - 127) code. A
pool is uint8 [blocks, bytes]; a block holds the codes [KV head][token][head_dim
bits / 8], then the bytes E [KV head][token][head_dim / 32].
"""
import math
import random

import torch

own = False

F32, F64 = torch.float32, torch.float64
GROUP = 32


# ------------------------------------------------------------------- cases --

def _case(name, kind, bits, n_seq, chunks, chunk, max_len, ragged, Hq, Hkv, d, bf16, page, mix, scaling="none"):
    return {"name": name, "kind": kind, "bits": bits, "n_seq": n_seq, "chunks": chunks, "chunk": chunk,
            "max_len": max_len, "ragged": ragged, "Hq": Hq, "Hkv": Hkv, "d": d, "bf16": bf16, "page": page, "mix": mix,
            "scaling": scaling}


def listed():
    return [
        # one generated token of each of a few sequences enters the cache
        _case("write4_decode", "write", 4, 16, 0, 1, 4096, True, 14, 2, 64, True, 16, 1),
        # chunks of long prompts beside generated tokens, positions scaled for
        # a long context
        _case("write4_chunks", "write", 4, 16, 4, 2048, 16384, True, 32, 8, 128, True, 16, 2, "yarn"),
        # chunks of odd lengths of a single-precision model, in 8 bits
        _case("write8_chunks_fp32", "write", 8, 7, 3, 777, 5000, True, 14, 2, 64, False, 32, 3, "linear"),
        # one sequence's cache as ordinary rows again (to be handed to a
        # prefill over contiguous rows)
        _case("read8_one", "read", 8, 1, 0, 1, 4096, False, 32, 4, 64, True, 16, 4),
        # many sequences of all lengths leave the cache
        _case("read4_many", "read", 4, 12, 0, 1, 16384, True, 32, 8, 128, True, 16, 5),
        # the prefill table's single token over a context of 4096
        _case("attend4_one", "attend", 4, 1, 0, 1, 4096, False, 32, 4, 64, True, 16, 6),
        # a serving step: one token of each of 64 sequences of all lengths
        _case("attend4_decode", "attend", 4, 64, 0, 1, 16384, True, 32, 8, 128, True, 16, 7),
        _case("attend8_decode", "attend", 8, 64, 0, 1, 16384, True, 32, 8, 128, True, 16, 7),
        # a few drafted tokens of each sequence are checked in one step
        _case("attend8_drafts", "attend", 8, 24, 24, 4, 8192, True, 32, 8, 128, True, 16, 8),
        # a late chunk of one long document
        _case("attend4_chunk_far", "attend", 4, 1, 1, 2048, 32768, False, 32, 8, 128, True, 16, 9),
        # chunks of four prompts in the same step as generated tokens
        _case("attend8_mixed", "attend", 8, 32, 4, 512, 8192, True, 14, 2, 64, True, 16, 10),
        # the same in single precision, with few sequences
        _case("attend4_mixed_fp32", "attend", 4, 8, 2, 500, 4096, True, 14, 2, 64, False, 16, 11),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(("write", "write", "read", "attend", "attend", "attend"))
    bf16 = rng.random() < 0.75
    d = 128 if bf16 and rng.random() < 0.5 else 64
    Hkv, group = rng.choice((1, 2, 4, 8)), rng.choice((1, 4, 7, 8))
    n_seq = _spread(rng, 1, 64)
    mode = "decode" if kind == "read" else rng.choice(("decode", "chunks", "mixed", "drafts"))
    chunks = {"decode": 0, "chunks": min(n_seq, 8), "mixed": (n_seq + 7) // 8, "drafts": n_seq}[mode]
    chunk = rng.randint(2, 8) if mode == "drafts" else _spread(rng, 2, 2048) if chunks else 1
    # the cache, what is read of it, and the scores of the chunks stay below
    # the largest listed case's
    most = int((3.2e8 if kind == "read" else 2.0e9) / (n_seq * Hkv * d * 4))
    if chunks:
        most = min(most, int(2.1e9 / (chunks * Hkv * group * chunk)))
    max_len = max(chunk, min(most, _spread(rng, 64, 32768)))
    return {"kind": kind, "bits": rng.choice((8, 4)), "n_seq": n_seq if mode != "chunks" else chunks, "chunks": chunks,
            "chunk": chunk, "max_len": max_len, "ragged": rng.random() < 0.8, "Hq": Hkv * group, "Hkv": Hkv, "d": d,
            "bf16": bf16, "page": rng.choice((16, 16, 32, 64, 128)), "mix": rng.randrange(1 << 20),
            "scaling": rng.choice(("none", "linear", "yarn"))}


def _lengths(case):
    """(new tokens, whole length) of each sequence, by the case alone; a read
    takes every position."""
    r = random.Random(case["mix"])
    got = []
    for s in range(case["n_seq"]):
        new = case["chunk"] if s < case["chunks"] else 1
        if case["ragged"]:
            new = r.randint((new + 1) // 2, new)
            whole = r.randint(max(new, case["max_len"] // 8), case["max_len"])
        else:
            whole = case["max_len"]
        got.append((whole if case["kind"] == "read" else new, whole))
    r.shuffle(got)
    return got


# -------------------------------------------------------------- the format --

def _scale_of(x, bits):
    """The bytes E of groups x [..., GROUP] in 32 bits: the least power of two by
    which the largest element is at most 448 (8 bits) or 7 (4 bits: from 6 on it
    rounds to 6), E at least 10 (also of zeros); 255 where one is not finite."""
    m, e = torch.frexp(x.abs().amax(-1))
    E = (e + (m > 0.875).to(e.dtype) - (9 if bits == 8 else 3) + 127).clamp(min=10)
    E = torch.where(m > 0.0, E, 10)
    return torch.where(torch.isfinite(x).all(-1), E, 255)


def _power(E):
    """2^(E - 127) in 32 bits."""
    return torch.where(E == 255, math.nan, torch.ldexp(torch.ones((), device=E.device), E - 127))


def _quantise(x, bits):
    """Rows x [..., d] in 32 bits: codes uint8 [..., d bits / 8] and E uint8 [..., d / 32]."""
    g = x.unflatten(-1, (-1, GROUP))
    E = _scale_of(g, bits)
    z = torch.where((E == 255)[..., None], 0.0, torch.ldexp(g, (127 - E)[..., None]))
    if bits == 8:
        codes = z.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8).flatten(-2)
    else:
        a = z.abs().clamp(max=6.0)
        step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0))
        a = torch.round(a / step) * step
        # 0, 0.5, 1, 1.5, 2, 3, 4, 6 are 0 to 7
        c = torch.where(a < 2.0, 2.0 * a, torch.where(a < 4.0, a + 2.0, 0.5 * a + 4.0)).to(torch.uint8)
        c = (c | (torch.signbit(z).to(torch.uint8) << 3)).flatten(-2)
        codes = c[..., 0::2] | (c[..., 1::2] << 4)
    return codes, E.to(torch.uint8)


def _values(codes, E, bits):
    """What codes and E stand for, in 32 bits."""
    if bits == 8:
        v = codes.view(torch.float8_e4m3fn).to(F32)
    else:
        c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
        i = (c & 7).to(F32)
        v = torch.where(i < 4.0, 0.5 * i, torch.where(i < 6.0, i - 2.0, 2.0 * i - 8.0))
        v = torch.where(c >= 8, -v, v)
    return (v.unflatten(-1, (-1, GROUP)) * _power(E.to(torch.int32))[..., None]).flatten(-2)


def _parts(pool, case):
    """A pool's codes and E as views [blocks, KV head, token, bytes]."""
    n, page, Hkv, d = pool.shape[0], case["page"], case["Hkv"], case["d"]
    cb, sb = d * case["bits"] // 8, d // GROUP
    codes = pool[:, :Hkv * page * cb].unflatten(1, (Hkv, page, cb))
    return codes, pool[:, Hkv * page * cb:Hkv * page * (cb + sb)].unflatten(1, (Hkv, page, sb))


def _block_bytes(case):
    n = case["Hkv"] * case["page"] * (case["d"] * case["bits"] // 8 + case["d"] // GROUP)
    return -(-n // 16) * 16


def _read_rows(pool, case, block, at):
    """The values [..., KV head, d] at tokens `at` of blocks `block`, in 32 bits."""
    codes, E = _parts(pool, case)
    return _values(codes[block, :, at], E[block, :, at], case["bits"])


# ------------------------------------------------------------------ inputs --

def _dtype(case):
    return torch.bfloat16 if case["bf16"] else F32


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _frequencies(dim, scaling):
    """The pairs' angles per position, in 64 bits, and the rotation's factor:
    base 10000, each divided by 4 ("linear"), or ("yarn") by up to 8 where a
    pair turns less than 32 times over 4096 positions, wholly where less than
    once."""
    f = 10000.0 ** (-torch.arange(0, dim, 2, dtype=F64, device="cuda") / dim)
    if scaling == "linear":
        return f / 4.0, 1.0
    if scaling == "yarn":
        def pair(turns):
            return dim * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(10000.0))
        lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), dim - 1)
        ramp = ((torch.arange(dim // 2, dtype=F64, device="cuda") - lo) / max(hi - lo, 0.001)).clamp_(0, 1)
        return f / 8.0 * ramp + f * (1 - ramp), 0.1 * math.log(8.0) + 1.0
    return f, 1.0


def _table(g, lens, page, spare):
    """Block tables of sequences of these lengths over a pool whose blocks are
    handed out in any order, and the pool's blocks."""
    need = [-(-n // page) for n in lens]
    n_blocks = sum(need) + spare
    order = torch.randperm(n_blocks, generator=g, device="cuda").to(torch.int32)
    wide = max(need)
    first = torch.tensor([0] + need[:-1], device="cuda").cumsum(0)
    col = torch.arange(wide, device="cuda")
    used = col[None, :] < torch.tensor(need, device="cuda")[:, None]
    table = torch.where(used, order[(first[:, None] + col[None, :]).clamp_(max=n_blocks - 1)], -1)
    return table.contiguous(), n_blocks


def _pool(g, case, n_blocks, spread):
    """A pool filled by rows whose channels are of sizes of their own, as keys
    have them (spread 0: all of one size)."""
    page, Hkv, d = case["page"], case["Hkv"], case["d"]
    pool = torch.zeros((n_blocks, _block_bytes(case)), dtype=torch.uint8, device="cuda")
    size = torch.exp(spread * torch.randn((Hkv, 1, d), generator=g, device="cuda"))
    codes, E = _parts(pool, case)
    step = max(1, (1 << 26) // (page * Hkv * d))
    for i in range(0, n_blocks, step):
        n = min(step, n_blocks - i)
        x = torch.randn((n, Hkv, page, d), generator=g, device="cuda").mul_(size)
        codes[i:i + n], E[i:i + n] = _quantise(x, case["bits"])
    return pool


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    st = {"case": case}
    Hq, Hkv, d, page = (case[x] for x in ("Hq", "Hkv", "d", "page"))
    dt = _dtype(case)
    st["lengths"] = pairs = _lengths(case)
    new, lens = [p[0] for p in pairs], [p[1] for p in pairs]
    ends = [sum(new[:i + 1]) for i in range(len(new))]
    st["cu_q"], st["lens"], st["max_new"] = _int([0] + ends), _int(lens), max(new)
    st["table"], n_blocks = _table(g, lens, page, 3 + len(lens) // 2)
    n_tok = sum(new)
    st["kc"], st["vc"] = _pool(g, case, n_blocks, 0.5), _pool(g, case, n_blocks, 0.0)
    if case["kind"] != "read":
        # Q, K and V of the new tokens, as a fused projection gives them
        st["qkv"] = torch.randn((n_tok, (Hq + 2 * Hkv) * d), generator=g, device="cuda").to(dt)
        st["out"] = torch.empty((n_tok, Hq * d), dtype=dt, device="cuda")
    if case["kind"] != "attend":
        st["k"], st["v"] = (torch.empty((n_tok, Hkv * d), dtype=dt, device="cuda") for _ in range(2))
    st["frequencies"], st["factor"] = _frequencies(d, case["scaling"])
    # the sequences by what they have, as a scheduler keeps them: several
    # tokens, single ones, and the longest of each
    for name, which in (("many", [s for s, p in enumerate(pairs) if p[0] > 1]),
                        ("one", [s for s, p in enumerate(pairs) if p[0] == 1])):
        st[name] = (torch.tensor(which, dtype=torch.long, device="cuda"), max([lens[s] for s in which], default=0))
    return st


# ---------------------------------------------------------- the plain forms --

def _places(st):
    """Position, block and token of the block of each row."""
    page = st["case"]["page"]
    tok = torch.arange(st["k"].shape[0], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(st["cu_q"][1:], tok, right=True)
    at = (st["lens"][seq] - st["cu_q"][seq + 1] + tok).long()
    return at, st["table"][seq, at // page].long(), at % page


def _turn(x, cos, sin):
    """Halves of x's rows turned by (cos, sin), in their type."""
    a, b = x.to(cos.dtype).chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _read_plain(st):
    case = st["case"]
    _, block, at = _places(st)
    for name, pool in (("k", "kc"), ("v", "vc")):
        # (the values are exact in either type)
        st[name].copy_(_read_rows(st[pool], case, block, at).flatten(-2))
    return {"k": st["k"], "v": st["v"]}


def _write_plain(st):
    case = st["case"]
    Hq, Hkv, d, bits = (case[x] for x in ("Hq", "Hkv", "d", "bits"))
    pos, block, at = _places(st)
    angle = pos.to(F64)[:, None, None] * st["frequencies"]
    cos, sin = angle.cos() * st["factor"], angle.sin() * st["factor"]
    q, k, v = st["qkv"].view(-1, Hq + 2 * Hkv, d).split([Hq, Hkv, Hkv], dim=1)
    st["out"].copy_(_turn(q, cos.to(F32), sin.to(F32)).flatten(1))
    # which code a key gets hangs on which side of a border it lies: in 64
    # bits, rounded to 32 for the quantiser
    for x, pool in ((_turn(k, cos, sin).to(F32), "kc"), (v.to(F32), "vc")):
        codes, E = _parts(st[pool], case)
        codes[block, :, at], E[block, :, at] = _quantise(x, bits)
    return {"q": st["out"]} | _read_plain(st)


def _attend_group(st, idx, longest, new):
    """Attention of the sequences `idx` (at most `new` new tokens each) in one
    padded batch, in 32 bits."""
    case = st["case"]
    Hq, Hkv, d, page = (case[x] for x in ("Hq", "Hkv", "d", "page"))
    G, m = Hq // Hkv, idx.numel()
    lens, first = st["lens"][idx].long(), st["cu_q"][idx].long()
    count = st["cu_q"][idx + 1].long() - first
    at = torch.arange(longest, device="cuda")
    block = st["table"][idx][:, at // page].long().clamp_(min=0)
    i = torch.arange(new, device="cuda")
    tok = first[:, None] + torch.minimum(i[None, :], count[:, None] - 1)
    q = st["qkv"][:, :Hq * d][tok].to(F32).view(m, new, Hkv, G, d).permute(0, 2, 3, 1, 4).reshape(m, Hkv, G * new, d)
    inside = (at % page).expand(m, -1)
    k = _read_rows(st["kc"], case, block, inside).permute(0, 2, 3, 1).contiguous()
    s = torch.matmul(q, k).mul_(1.0 / math.sqrt(d)).view(m, Hkv, G, new, longest)
    del k
    position = lens[:, None] - count[:, None] + torch.minimum(i[None, :], count[:, None] - 1)
    s.masked_fill_((at[None, None, :] > position[:, :, None])[:, None, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    total = s.sum(-1, keepdim=True)
    v = _read_rows(st["vc"], case, block, inside).transpose(1, 2).contiguous()
    o = torch.matmul(s.view(m, Hkv, G * new, longest), v).view(m, Hkv, G, new, d) / total
    # a padded row is the sequence's last one again
    st["out"][tok.view(-1)] = o.permute(0, 3, 1, 2, 4).reshape(m * new, Hq * d).to(st["out"].dtype)


def _attend_plain(st):
    # a chunk's padding would multiply the generated tokens' work: two batches
    if st["many"][1]:
        _attend_group(st, *st["many"], st["max_new"])
    if st["one"][1]:
        _attend_group(st, *st["one"], 1)
    return {"out": st["out"]}


# ----------------------------------------------------------------- one pass --

def run(st):
    case = st["case"]
    kind = case["kind"]
    if not own:
        return _write_plain(st) if kind == "write" else _read_plain(st) if kind == "read" else _attend_plain(st)
    import mx230_amd as mx
    pages = (st["table"], case["page"], st["cu_q"], st["lens"])
    if kind == "attend":
        mx.run_prefill_batch_mx(st["qkv"], st["kc"], st["vc"], case["bits"], st["out"], *pages, st["max_new"],
                                case["Hq"], case["Hkv"], case["d"])
        return {"out": st["out"]}
    got = {}
    if kind == "write":
        mx.run_cache_append_mx(st["qkv"], st["out"], st["kc"], st["vc"], case["bits"], *pages, case["Hq"], case["Hkv"],
                               case["d"], frequencies=st["frequencies"], factor=st["factor"])
        got["q"] = st["out"]
    mx.run_cache_read_mx(st["kc"], st["vc"], case["bits"], st["k"], st["v"], *pages, case["Hkv"], case["d"])
    return got | {"k": st["k"], "v": st["v"]}


def work(case):
    es = 2 if case["bf16"] else 4
    Hq, Hkv, d = case["Hq"], case["Hkv"], case["d"]
    held = d * case["bits"] // 8 + d // GROUP  # bytes of a head's row in the cache
    pairs = _lengths(case)
    n_tok = sum(new for new, _ in pairs)
    if case["kind"] == "read":
        return {"bytes": n_tok * 2 * Hkv * (held + d * es), "flops": n_tok * 2 * Hkv * d}
    if case["kind"] == "write":
        # qkv in, q out, the new rows written and read, and their values out
        return {"bytes": n_tok * (es * d * (2 * Hq + 4 * Hkv) + 4 * Hkv * held),
                "flops": 3 * n_tok * (Hq + Hkv) * d + 4 * n_tok * Hkv * d}
    seen = sum(n * ln - n * (n - 1) // 2 for n, ln in pairs)
    blocks = sum(-(-ln // case["page"]) for _, ln in pairs)
    return {"bytes": 2 * es * d * n_tok * Hq + 2 * Hkv * held * sum(ln for _, ln in pairs) + 4 * blocks,
            "flops": 4.0 * seen * Hq * d}


# --------------------------------------------------------------- in 64 bits --

def _levels(bits):
    """The values of the non-negative codes, by code."""
    man, bias, n = (3, 7, 127) if bits == 8 else (1, 1, 8)
    return torch.tensor([(c % (1 << man)) * 2.0 ** (1 - bias - man) if c >> man == 0 else
                         (1 + (c % (1 << man)) * 2.0 ** -man) * 2.0 ** ((c >> man) - bias) for c in range(n)],
                        dtype=F64, device="cuda")


def _stands_for(x, bits):
    """x [..., d] in 64 bits as the cache holds it: the nearest of the levels, on
    a tie the even code's."""
    lv, top = _levels(bits), 448.0 if bits == 8 else 7.0
    g = x.unflatten(-1, (-1, GROUP))
    most = g.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(most / top)).clamp(min=-117.0)
    e = torch.where(most > top * torch.exp2(e), e + 1, e)
    e = torch.where((most <= top * torch.exp2(e - 1)) & (e > -117.0), e - 1, e)
    z = g * torch.exp2(-e)
    a = z.abs().clamp(max=float(lv[-1])).contiguous()
    hi = torch.searchsorted(lv, a).clamp(1, lv.numel() - 1)
    down, up = a - lv[hi - 1], lv[hi] - a
    c = torch.where((down < up) | ((down == up) & (hi % 2 == 1)), hi - 1, hi)
    return (torch.copysign(lv[c], z) * torch.exp2(e)).flatten(-2)


def _held(pool, case, block, at, h):
    """KV head h's values at tokens `at` of blocks `block`, in 64 bits, by table."""
    codes, E = _parts(pool, case)
    c, E = codes[block, h, at].long(), E[block, h, at].to(F64)
    lv = _levels(case["bits"])
    if case["bits"] == 4:
        c = torch.stack([c % 16, c // 16], -1).flatten(-2)
        lv = torch.cat([lv, -lv])
    else:
        lv = torch.cat([lv, torch.full((1,), math.nan, dtype=F64, device="cuda")])
        lv = torch.cat([lv, -lv])
    return lv[c] * torch.exp2(E - 127.0).repeat_interleave(GROUP, -1)


def exact(case, seed):
    st = prepare(case, seed)
    Hq, Hkv, d, page, bits = (case[x] for x in ("Hq", "Hkv", "d", "page", "bits"))
    n_tok, t0 = sum(new for new, _ in st["lengths"]), 0
    q = torch.empty((n_tok, Hq * d), dtype=F64, device="cuda")
    k, v = (torch.empty((n_tok, Hkv, d), dtype=F64, device="cuda") for _ in range(2))
    for s, (new, ln) in enumerate(st["lengths"]):
        at = torch.arange(ln, device="cuda")
        block, inside = st["table"][s].long()[at // page], at % page
        rows = slice(t0, t0 + new)
        if case["kind"] == "write":
            mine = st["qkv"][rows].to(F64).view(new, Hq + 2 * Hkv, d)
            turn = torch.polar(torch.full((new, 1, d // 2), st["factor"], dtype=F64, device="cuda"),
                               at[ln - new:].to(F64)[:, None, None] * st["frequencies"])
            z = torch.complex(mine[:, :Hq + Hkv, :d // 2], mine[:, :Hq + Hkv, d // 2:]) * turn
            turned = torch.cat([z.real, z.imag], -1)
            q[rows] = turned[:, :Hq].reshape(new, Hq * d)
            k[rows], v[rows] = _stands_for(turned[:, Hq:], bits), _stands_for(mine[:, Hq + Hkv:], bits)
        elif case["kind"] == "read":
            for h in range(Hkv):
                k[rows, h], v[rows, h] = (_held(st[x], case, block, inside, h) for x in ("kc", "vc"))
        else:
            mine = st["qkv"][rows, :Hq * d].to(F64).view(new, Hq, d)
            for h in range(Hkv):
                ks, vs = (_held(st[x], case, block, inside, h) for x in ("kc", "vc"))
                for j in range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv)):
                    for i in range(0, new, 1024):
                        n = min(1024, new - i)
                        p = (mine[i:i + n, j] @ ks.T) / math.sqrt(d)
                        p.masked_fill_(at[None, :] > at[ln - new + i:ln - new + i + n, None], -math.inf)
                        q[t0 + i:t0 + i + n, j * d:(j + 1) * d] = torch.softmax(p, 1) @ vs
        t0 += new
    if case["kind"] == "attend":
        return {"out": q}
    got = {"k": k.flatten(1), "v": v.flatten(1)}
    return got if case["kind"] == "read" else {"q": q} | got
