"""The operators around attention over a paged cache, as measurable cases.

Four operators: rotary positions (training, forward and gradient), the rotary
write of new tokens into a paged cache, attention of a batch of sequences' new
tokens over that cache, and the upkeep of its pages (fork, free, compact). Each
listed case stands for a use named at its entry; draw() gives more of the same
ranges.
"""
import math
import random

import torch

own = False

F32, F64 = torch.float32, torch.float64


# ------------------------------------------------------------------- cases --

def _rotary(name, B, Hq, Hkv, N, d, dim, interleaved, scaling, bf16, packed):
    return {"name": name, "kind": "rotary", "B": B, "Hq": Hq, "Hkv": Hkv, "N": N, "d": d, "dim": dim,
            "interleaved": interleaved, "scaling": scaling, "bf16": bf16, "packed": packed}


def _batch(name, kind, n_seq, chunks, chunk, max_len, ragged, Hq, Hkv, d, bf16, page, mix, scaling="none"):
    return {"name": name, "kind": kind, "n_seq": n_seq, "chunks": chunks, "chunk": chunk, "max_len": max_len,
            "ragged": ragged, "Hq": Hq, "Hkv": Hkv, "d": d, "bf16": bf16, "page": page, "mix": mix,
            "scaling": scaling}


def _fork(name, parents, fan, max_len, pools, width, page, mix):
    return {"name": name, "kind": "fork", "parents": parents, "fan": fan, "max_len": max_len, "pools": pools,
            "width": width, "page": page, "mix": mix}


def _compact(name, n_blocks, live, moves, n_seq, pools, width, page):
    return {"name": name, "kind": "compact", "n_blocks": n_blocks, "live": live, "moves": moves, "n_seq": n_seq,
            "pools": pools, "width": width, "page": page}


def listed():
    return [
        # the benchmark's training step: rotary positions before its attention
        _rotary("rotary_train", 4, 12, 12, 4096, 64, 64, False, "none", True, False),
        # short single-precision rows of odd length, half of each head rotated
        # in neighbouring pairs, several documents packed into a row
        _rotary("rotary_packed_fp32", 3, 10, 10, 777, 64, 32, True, "linear", False, True),
        # one generated token of each of a few sequences enters the cache
        _batch("append_decode", "append", 16, 0, 1, 4096, True, 14, 2, 64, True, 16, 1),
        # chunks of long prompts beside generated tokens, positions scaled for
        # a long context
        _batch("append_chunks", "append", 16, 4, 2048, 16384, True, 32, 8, 128, True, 16, 2, "yarn"),
        # the prefill table's single token over a context of 4096
        _batch("attend_one", "attend", 1, 0, 1, 4096, False, 32, 4, 64, True, 16, 3),
        # a serving step: one token of each of 64 sequences of all lengths
        _batch("attend_decode", "attend", 64, 0, 1, 16384, True, 32, 8, 128, True, 16, 4),
        # a late chunk of one long document
        _batch("attend_chunk_far", "attend", 1, 1, 2048, 32768, False, 32, 8, 128, True, 16, 5),
        # chunks of four prompts in the same step as generated tokens
        _batch("attend_mixed", "attend", 32, 4, 512, 8192, True, 14, 2, 64, True, 16, 6),
        # the same in single precision, with few sequences
        _batch("attend_mixed_fp32", "attend", 8, 2, 500, 4096, True, 14, 2, 64, False, 16, 7),
        # one beam step of a single small request
        _fork("fork_small", 1, 4, 1000, 2, 128, 16, 8),
        # a beam step of 8 requests of 8 beams over 24 layers' caches
        _fork("fork_beams", 8, 8, 4096, 48, 128, 16, 9),
        # a pool after many requests have come and gone, moved to its low end
        _compact("compact", 8192, 5000, 2000, 48, 8, 1024, 16),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _lengths(case):
    """(new tokens, whole length) of each sequence, by the case alone."""
    r = random.Random(case["mix"])
    got = []
    for s in range(case["n_seq"]):
        new = case["chunk"] if s < case["chunks"] else 1
        if case["ragged"]:
            new = r.randint((new + 1) // 2, new)
            got.append((new, r.randint(max(new, case["max_len"] // 8), case["max_len"])))
        else:
            got.append((new, case["max_len"]))
    r.shuffle(got)
    return got


def draw(rng):
    u = rng.random()
    if u < 0.2:
        bf16 = rng.random() < 0.6
        d = rng.choice((64, 128))
        Hkv, group = rng.choice((1, 2, 3, 4, 8)), rng.choice((1, 1, 4, 7, 8))
        N = _spread(rng, 16, 8192)
        # no more bytes than the training step of the benchmark
        B = rng.randint(1, max(1, min(8, int(25e6 / ((Hkv + Hkv * group) * N * d * (1 if bf16 else 2))))))
        return {"kind": "rotary", "B": B, "Hq": Hkv * group, "Hkv": Hkv, "N": N, "d": d,
                "dim": rng.choice((d, d, d // 2, d // 4, 24)), "interleaved": rng.random() < 0.4,
                "scaling": rng.choice(("none", "linear", "yarn")), "bf16": bf16, "packed": rng.random() < 0.4}
    if u < 0.8:
        attend = u >= 0.4
        bf16 = rng.random() < 0.75
        d = 128 if bf16 and rng.random() < 0.5 else 64
        Hkv, group = rng.choice((1, 2, 4, 8)), rng.choice((1, 4, 7, 8))
        n_seq = _spread(rng, 1, 64)
        mode = rng.choice(("decode", "chunks", "mixed"))
        chunks = 0 if mode == "decode" else min(n_seq, 8) if mode == "chunks" else (n_seq + 7) // 8
        chunk = _spread(rng, 2, 2048) if chunks else 1
        # the cache, and the scores of the chunks, stay below the largest listed case's
        most = int(2.0e9 / (n_seq * Hkv * d * 4))
        if chunks:
            most = min(most, int(2.1e9 / (chunks * Hkv * group * chunk)))
        max_len = max(chunk, min(most, _spread(rng, 64, 32768)))
        return {"kind": "attend" if attend else "append", "n_seq": n_seq if mode != "chunks" else chunks,
                "chunks": chunks, "chunk": chunk, "max_len": max_len, "ragged": rng.random() < 0.8,
                "Hq": Hkv * group, "Hkv": Hkv, "d": d, "bf16": bf16, "page": rng.choice((16, 16, 32, 64, 128)),
                "mix": rng.randrange(1 << 20), "scaling": rng.choice(("none", "linear", "yarn"))}
    width = rng.choice((64, 128, 256, 1024))
    page = rng.choice((16, 32, 64))
    if u < 0.9:
        parents, fan = _spread(rng, 1, 16), rng.randint(1, 8)
        max_len = _spread(rng, 40, 4096)
        pools = _spread(rng, 1, max(1, min(48, int(4e8 / (parents * (2 * fan + 2) * (max_len + page) * width)))))
        return {"kind": "fork", "parents": parents, "fan": fan, "max_len": max_len, "pools": pools, "width": width,
                "page": page, "mix": rng.randrange(1 << 20)}
    n_blocks = _spread(rng, 100, 16384)
    live = rng.randint(n_blocks // 3, n_blocks * 2 // 3)
    pools = _spread(rng, 1, max(1, min(48, int(1.0e9 / (n_blocks * page * width)))))
    return {"kind": "compact", "n_blocks": n_blocks, "live": live,
            "moves": rng.randint(1, min(live, n_blocks - live)), "n_seq": rng.randint(1, min(64, live // 8)),
            "pools": pools, "width": width, "page": page}


# ------------------------------------------------------------------ inputs --

def _dtype(case):
    return torch.bfloat16 if case["bf16"] else F32


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, shape, dtype, scale=1.0):
    t = torch.empty(shape, dtype=dtype, device="cuda")
    flat = t.view(-1)
    for part in flat.split(1 << 28):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda").mul_(scale))
    return t


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


def _tables(g, lens, page, spare):
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


def prepare(case, seed):
    g = _gen(seed)
    st = {"case": case}
    if case["kind"] == "rotary":
        B, Hq, Hkv, N, d = (case[x] for x in ("B", "Hq", "Hkv", "N", "d"))
        dt = _dtype(case)
        st["frequencies"], st["factor"] = _frequencies(case["dim"], case["scaling"])
        # views of a fused projection's rows, as an attention block has them
        qkv = _randn(g, (B, N, Hq + 2 * Hkv, d), dt)
        st["q"] = qkv[:, :, :Hq].transpose(1, 2).requires_grad_(True)
        st["k"] = qkv[:, :, Hq:Hq + Hkv].transpose(1, 2).requires_grad_(True)
        # gradients come from the attention's backward, packed per head
        st["dq"], st["dk"] = _randn(g, (B, Hq, N, d), dt, 0.02), _randn(g, (B, Hkv, N, d), dt, 0.02)
        st["positions"] = None
        if case["packed"]:
            # documents of random lengths one after another: positions start over
            starts = torch.rand((B, N), generator=g, device="cuda") < 8.0 / N
            at = torch.arange(N, device="cuda")[None, :].expand(B, N)
            st["positions"] = (at - torch.where(starts, at, 0).cummax(1).values).to(torch.int32).contiguous()
    elif case["kind"] in ("append", "attend"):
        Hq, Hkv, d, page = (case[x] for x in ("Hq", "Hkv", "d", "page"))
        dt = _dtype(case)
        st["lengths"] = pairs = _lengths(case)
        new, lens = [p[0] for p in pairs], [p[1] for p in pairs]
        ends = [sum(new[:i + 1]) for i in range(len(new))]
        st["cu_q"], st["lens"], st["max_new"] = _int([0] + ends), _int(lens), max(new)
        st["table"], n_blocks = _tables(g, lens, page, 3 + len(lens) // 2)
        n_tok = sum(new)
        # Q, K and V of the new tokens, as a fused projection gives them
        st["qkv"] = _randn(g, (n_tok, (Hq + 2 * Hkv) * d), dt)
        st["kc"], st["vc"] = (_randn(g, (n_blocks * page, Hkv * d), dt) for _ in range(2))
        st["out"] = torch.empty((n_tok, Hq * d), dtype=dt, device="cuda")
        st["frequencies"], st["factor"] = _frequencies(d, case["scaling"])
        # the sequences by what they have, as a scheduler keeps them: chunks,
        # single tokens, and the longest of each
        for name, which in (("many", [s for s, p in enumerate(pairs) if p[0] > 1]),
                            ("one", [s for s, p in enumerate(pairs) if p[0] == 1])):
            st[name] = (torch.tensor(which, dtype=torch.long, device="cuda"), max([lens[s] for s in which], default=0))
    elif case["kind"] == "fork":
        r = random.Random(case["mix"])
        n, fan, page = case["parents"], case["fan"], case["page"]
        st["lengths"] = lens = [r.randint(case["max_len"] // 2, case["max_len"]) for _ in range(n)]
        # each parent's beams hold sequences of their own, which end now
        ended = [r.randint(1, case["max_len"]) for _ in range(n * fan)]
        st["table"], st["n_blocks"] = _tables(g, lens + ended, page, n * fan)
        st["lens"] = _int(lens + ended)
        st["refs"] = torch.zeros(st["n_blocks"], dtype=torch.int32, device="cuda")
        held = st["table"].reshape(-1)
        st["refs"].index_add_(0, held.clamp(min=0).long(), (held >= 0).to(torch.int32))
        st["parents"] = _int([i // fan for i in range(n * fan)])
        st["children"] = _int([n + i for i in range(n * fan)])
        st["pools"] = _randn(g, (case["pools"], st["n_blocks"] * page, case["width"]), torch.bfloat16)
        st["pairs"] = torch.empty((n * fan, 2), dtype=torch.int32, device="cuda")
        st["status"] = torch.empty(n * fan, dtype=torch.int32, device="cuda")
        st["counts"] = torch.empty(2, dtype=torch.int32, device="cuda")
        st["copied"] = torch.tensor([i for i in range(n * fan) if lens[i // fan] % page], dtype=torch.long, device="cuda")
    else:
        n_blocks, live, moves, n_seq, page = (case[x] for x in ("n_blocks", "live", "moves", "n_seq", "page"))
        # `moves` free blocks among the first `live`, as many used ones behind
        low = torch.randperm(live, generator=g, device="cuda")[:live - moves]
        high = live + torch.randperm(n_blocks - live, generator=g, device="cuda")[:moves]
        blocks = torch.cat([low, high])[torch.randperm(live, generator=g, device="cuda")]
        wide = -(-live // n_seq)
        table = torch.full((n_seq * wide,), -1, dtype=torch.int32, device="cuda")
        table[:live] = blocks.to(torch.int32)
        st["table"] = table.view(n_seq, wide)
        full = [min(wide, max(0, live - i * wide)) for i in range(n_seq)]
        st["lens"] = _int([max(0, x * page - (3 * i) % page) for i, x in enumerate(full)])
        st["refs"] = torch.zeros(n_blocks, dtype=torch.int32, device="cuda")
        st["refs"][blocks] = 1
        st["pools"] = _randn(g, (case["pools"], n_blocks * page, case["width"]), torch.bfloat16)
        st["new_table"], st["new_refs"] = torch.empty_like(st["table"]), torch.empty_like(st["refs"])
        st["pairs"] = torch.empty((max(1, n_blocks // 2), 2), dtype=torch.int32, device="cuda")
        st["counts"] = torch.empty(2, dtype=torch.int32, device="cuda")
    return st


# ---------------------------------------------------------- the plain forms --

def _turn(x, cos, sin, interleaved):
    """Pairs of x's first elements turned by (cos, sin), in 32 bits, rounded once."""
    dim = 2 * cos.shape[-1]
    y = x.to(F32, copy=True)
    if interleaved:
        a, b = y[..., 0:dim:2].clone(), y[..., 1:dim:2].clone()
        y[..., 0:dim:2], y[..., 1:dim:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = y[..., :dim // 2].clone(), y[..., dim // 2:dim].clone()
        y[..., :dim // 2], y[..., dim // 2:dim] = a * cos - b * sin, b * cos + a * sin
    return y.to(x.dtype)


def _angles(positions, st):
    """cos and sin of positions x frequencies: the angles in 64 bits."""
    a = positions.to(F64)[..., None] * st["frequencies"]
    return (a.cos() * st["factor"]).to(F32), (a.sin() * st["factor"]).to(F32)


def _rotary_plain(st):
    case = st["case"]
    at = st["positions"] if st["positions"] is not None else torch.arange(case["N"], device="cuda")[None, :]
    cos, sin = (t[:, None] for t in _angles(at, st))
    il = case["interleaved"]
    return {"q": _turn(st["q"].detach(), cos, sin, il), "k": _turn(st["k"].detach(), cos, sin, il),
            "dq": _turn(st["dq"], cos, -sin, il), "dk": _turn(st["dk"], cos, -sin, il)}


def _append_plain(st):
    case = st["case"]
    Hq, Hkv, d, page = (case[x] for x in ("Hq", "Hkv", "d", "page"))
    qkv = st["qkv"]
    n = qkv.shape[0]
    tok = torch.arange(n, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(st["cu_q"][1:], tok, right=True)
    at = (st["lens"][seq] - st["cu_q"][seq + 1] + tok).long()
    row = st["table"][seq, at // page].long() * page + at % page
    cos, sin = (t[:, None] for t in _angles(at, st))
    q, k, v = qkv.view(n, Hq + 2 * Hkv, d).split([Hq, Hkv, Hkv], dim=1)
    st["out"].copy_(_turn(q, cos, sin, False).reshape(n, Hq * d))
    st["kc"][row] = _turn(k, cos, sin, False).reshape(n, Hkv * d)
    st["vc"][row] = v.reshape(n, Hkv * d)
    return {"q": st["out"], "kc": st["kc"], "vc": st["vc"]}


def _attend_group(st, idx, longest, new):
    """Attention of the sequences `idx` (at most `new` new tokens each) in one
    padded batch, in 32 bits."""
    case = st["case"]
    Hq, Hkv, d, page = (case[x] for x in ("Hq", "Hkv", "d", "page"))
    G, m = Hq // Hkv, idx.numel()
    lens, first = st["lens"][idx].long(), st["cu_q"][idx].long()
    count = st["cu_q"][idx + 1].long() - first
    at = torch.arange(longest, device="cuda")
    row = st["table"][idx][:, at // page].long().clamp_(min=0) * page + at % page
    i = torch.arange(new, device="cuda")
    tok = first[:, None] + torch.minimum(i[None, :], count[:, None] - 1)
    q = st["qkv"][:, :Hq * d][tok].to(F32).view(m, new, Hkv, G, d).permute(0, 2, 3, 1, 4).reshape(m, Hkv, G * new, d)
    k = st["kc"][row].to(F32).view(m, longest, Hkv, d).permute(0, 2, 3, 1).contiguous()
    s = torch.matmul(q, k).mul_(1.0 / math.sqrt(d)).view(m, Hkv, G, new, longest)
    position = lens[:, None] - count[:, None] + torch.minimum(i[None, :], count[:, None] - 1)
    s.masked_fill_((at[None, None, :] > position[:, :, None])[:, None, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    total = s.sum(-1, keepdim=True)
    v = st["vc"][row].to(F32).view(m, longest, Hkv, d).permute(0, 2, 1, 3).contiguous()
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


def _copy_blocks(st, src, dst):
    pools = st["pools"]
    blocks = pools.view(pools.shape[0], -1, st["case"]["page"] * st["case"]["width"])
    blocks[:, dst] = blocks[:, src]


def _fork_plain(st):
    page, table, lens, refs = st["case"]["page"], st["table"], st["lens"], st["refs"]
    parents, children = st["parents"].long(), st["children"].long()
    # the ended sequences' blocks go back
    held = table[children].reshape(-1)
    refs.index_add_(0, held.clamp(min=0).long(), -(held >= 0).to(torch.int32))
    # the children take their parents' rows; a block that is not full is copied
    table[children] = table[parents]
    lens[children] = lens[parents]
    held = table[children].reshape(-1)
    refs.index_add_(0, held.clamp(min=0).long(), (held >= 0).to(torch.int32))
    pick = st["copied"]
    k = pick.numel()
    if k:
        last = lens[children[pick]].long() // page
        src = table[children[pick], last]
        dst = torch.argsort((refs != 0).to(torch.int8), stable=True)[:k]
        refs.index_add_(0, src.long(), torch.full((k,), -1, dtype=torch.int32, device="cuda"))
        refs[dst] = 1
        table[children[pick], last] = dst.to(torch.int32)
        _copy_blocks(st, src.long(), dst)
    return {"table": table, "lens": lens, "refs": refs, "pools": st["pools"]}


def _compact_plain(st):
    refs, table, moves = st["refs"], st["table"], st["case"]["moves"]
    n = refs.numel()
    at = torch.arange(n, device="cuda")
    used = refs > 0
    live = used.sum()
    dst = torch.argsort((used | (at >= live)).to(torch.int8), stable=True)[:moves]
    src = torch.argsort((~used | (at < live)).to(torch.int8), stable=True)[:moves]
    to = at.clone()
    to[src] = dst
    st["new_table"].copy_(torch.where(table >= 0, to[table.clamp(min=0).long()].to(torch.int32), table))
    st["new_refs"].copy_(refs)
    st["new_refs"][dst] = refs[src]
    st["new_refs"][src] = 0
    _copy_blocks(st, src, dst)
    return {"table": st["new_table"], "refs": st["new_refs"], "pools": st["pools"]}


# ----------------------------------------------------------------- one pass --

def run(st):
    case = st["case"]
    kind = case["kind"]
    if not own:
        if kind == "rotary":
            return _rotary_plain(st)
        if kind == "append":
            return _append_plain(st)
        if kind == "attend":
            return _attend_plain(st)
        return _fork_plain(st) if kind == "fork" else _compact_plain(st)
    import mx230_amd as mx
    if kind == "rotary":
        from mx230_amd.autograd import rotary_embedding
        q, k = rotary_embedding(st["q"], st["k"], st["frequencies"], positions=st["positions"],
                                interleaved=case["interleaved"], factor=st["factor"])
        dq, dk = torch.autograd.grad((q, k), (st["q"], st["k"]), (st["dq"], st["dk"]))
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    if kind == "append":
        mx.run_cache_append(st["qkv"], st["out"], st["kc"], st["vc"], st["table"], case["page"], st["cu_q"], st["lens"],
                            case["Hq"], case["Hkv"], case["d"], frequencies=st["frequencies"], factor=st["factor"])
        return {"q": st["out"], "kc": st["kc"], "vc": st["vc"]}
    if kind == "attend":
        mx.run_prefill_batch(st["qkv"], st["kc"], st["vc"], st["out"], st["table"], case["page"], st["cu_q"],
                             st["lens"], st["max_new"], case["Hq"], case["Hkv"], case["d"])
        return {"out": st["out"]}
    if kind == "fork":
        mx.run_pages_free(st["table"], case["page"], st["lens"], st["refs"], st["children"])
        mx.run_pages_fork(st["table"], case["page"], st["lens"], st["refs"], st["parents"], st["children"],
                          st["pairs"], st["status"], st["counts"])
        mx.run_pages_copy(st["pools"], case["page"], st["pairs"], st["counts"])
        return {"table": st["table"], "lens": st["lens"], "refs": st["refs"], "pools": st["pools"]}
    mx.run_pages_compact(st["table"], case["page"], st["lens"], st["refs"], st["new_table"], st["new_refs"],
                         st["pairs"], st["counts"])
    mx.run_pages_copy(st["pools"], case["page"], st["pairs"], st["counts"])
    return {"table": st["new_table"], "refs": st["new_refs"], "pools": st["pools"]}


def work(case):
    if case["kind"] == "rotary":
        es = 2 if case["bf16"] else 4
        n = case["B"] * case["N"] * (case["Hq"] + case["Hkv"])
        # each direction reads and writes whole heads; 4 products and 2 sums a pair
        return {"bytes": 4 * n * case["d"] * es, "flops": 2 * 3 * n * case["dim"]}
    if case["kind"] in ("append", "attend"):
        es = 2 if case["bf16"] else 4
        Hq, Hkv, d = case["Hq"], case["Hkv"], case["d"]
        pairs = _lengths(case)
        n_tok = sum(new for new, _ in pairs)
        if case["kind"] == "append":
            return {"bytes": 2 * n_tok * (Hq + 2 * Hkv) * d * es, "flops": 3 * n_tok * (Hq + Hkv) * d}
        seen = sum(n * ln - n * (n - 1) // 2 for n, ln in pairs)
        blocks = sum(-(-ln // case["page"]) for _, ln in pairs)
        return {"bytes": es * d * (2 * n_tok * Hq + 2 * Hkv * sum(ln for _, ln in pairs)) + 4 * blocks,
                "flops": 4.0 * seen * Hq * d}
    block = 2 * case["page"] * case["width"] * case["pools"]
    if case["kind"] == "fork":
        r = random.Random(case["mix"])
        page, fan = case["page"], case["fan"]
        lens = [r.randint(case["max_len"] // 2, case["max_len"]) for _ in range(case["parents"])]
        # a partly filled block is read and written per child, its table row
        # read and written and the row's counts raised; the ended rows' freed
        rows = sum(-(-n // page) for n in lens) * fan
        return {"bytes": 2 * block * fan * sum(1 for n in lens if n % page) + 32 * rows, "flops": 0}
    return {"bytes": 2 * block * case["moves"] + 8 * case["n_blocks"] + 8 * case["live"], "flops": 0}


# --------------------------------------------------------------- in 64 bits --

def _turned(x, positions, st, interleaved, sign=1.0):
    """x [..., n, d] at positions [..., n], pair by pair as complex numbers."""
    dim = 2 * st["frequencies"].numel()
    y = x.detach().to(F64).clone()
    turn = torch.polar(torch.full((), st["factor"], dtype=F64, device="cuda").expand(positions.shape + (dim // 2,)),
                       sign * positions.to(F64)[..., None] * st["frequencies"])
    if interleaved:
        z = torch.view_as_complex(y[..., :dim].reshape(y.shape[:-1] + (dim // 2, 2)).contiguous()) * turn
        y[..., :dim] = torch.view_as_real(z).reshape(y.shape[:-1] + (dim,))
    else:
        z = torch.complex(y[..., :dim // 2], y[..., dim // 2:dim]) * turn
        y[..., :dim // 2], y[..., dim // 2:dim] = z.real, z.imag
    return y


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "rotary":
        at = st["positions"]
        if at is None:
            at = torch.arange(case["N"], device="cuda").expand(case["B"], -1)
        at, il = at[:, None, :], case["interleaved"]
        return {"q": _turned(st["q"], at, st, il), "k": _turned(st["k"], at, st, il),
                "dq": _turned(st["dq"], at, st, il, -1.0), "dk": _turned(st["dk"], at, st, il, -1.0)}
    if kind in ("append", "attend"):
        Hq, Hkv, d, page = (case[x] for x in ("Hq", "Hkv", "d", "page"))
        G, t0 = Hq // Hkv, 0
        out = torch.empty(st["out"].shape, dtype=F64, device="cuda")
        kc, vc = (st[x].to(F64) if kind == "append" else st[x] for x in ("kc", "vc"))
        for s, (new, ln) in enumerate(st["lengths"]):
            at = torch.arange(ln, device="cuda")
            row = st["table"][s].long()[at // page] * page + at % page
            mine = st["qkv"][t0:t0 + new].to(F64).view(new, Hq + 2 * Hkv, d).transpose(0, 1)
            if kind == "append":
                turned = _turned(mine[:Hq + Hkv], at[ln - new:], st, False)
                out[t0:t0 + new] = turned[:Hq].transpose(0, 1).reshape(new, Hq * d)
                kc[row[ln - new:]] = turned[Hq:].transpose(0, 1).reshape(new, Hkv * d)
                vc[row[ln - new:]] = mine[Hq + Hkv:].transpose(0, 1).reshape(new, Hkv * d)
            else:
                ks, vs = kc[row].to(F64), vc[row].to(F64)
                for h in range(Hq):
                    c = slice(h // G * d, (h // G + 1) * d)
                    for i in range(0, new, 1024):
                        j = min(new, i + 1024)
                        p = (mine[h, i:j] @ ks[:, c].T) / math.sqrt(d)
                        p.masked_fill_(at[None, :] > at[ln - new + i:ln - new + j, None], -math.inf)
                        out[t0 + i:t0 + j, h * d:(h + 1) * d] = torch.softmax(p, 1) @ vs[:, c]
            t0 += new
        return {"out": out} if kind == "attend" else {"q": out, "kc": kc, "vc": vc}
    page = case["page"]
    table, lens, refs = (st[x].tolist() for x in ("table", "lens", "refs"))
    moved = []
    if kind == "fork":
        parents, children = st["parents"].tolist(), st["children"].tolist()
        for c in children:
            for j in range(-(-lens[c] // page)):
                refs[table[c][j]] -= 1
        free = iter([b for b, n in enumerate(refs) if n == 0])
        for p, c in zip(parents, children):
            full, lens[c] = lens[p] // page, lens[p]
            table[c] = table[p][:full] + [-1] * (len(table[p]) - full)
            for b in table[c][:full]:
                refs[b] += 1
            if lens[p] % page:
                b = next(free)
                table[c][full], refs[b] = b, 1
                moved.append((table[p][full], b))
    else:
        live = sum(1 for n in refs if n)
        moved = list(zip([b for b, n in enumerate(refs) if n and b >= live], [b for b, n in enumerate(refs) if not n]))
        to = dict(moved)
        table = [[to.get(b, b) for b in r] for r in table]
        for a, b in moved:
            refs[a], refs[b] = 0, refs[a]
    pools = st["pools"].clone()
    blocks = pools.view(pools.shape[0], -1, page * case["width"])
    if moved:
        blocks[:, torch.tensor([b for _, b in moved], device="cuda")] = \
            st["pools"].view_as(blocks)[:, torch.tensor([a for a, _ in moved], device="cuda")]
    whole = {"table": _int(table), "refs": _int(refs), "pools": pools}
    return whole | {"lens": _int(lens)} if kind == "fork" else whole
