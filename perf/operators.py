"""Cases of the operators for several continuations of a sequence on one KV cache: writing rows (head norm, rotation,
quantising), attention for drafted trees and single tokens over a binary16 or 8-bit cache, beam selection, and moving cached
rows.  ``run`` is one pass of a case, in elementary torch operations or, with ``own``, through ``blackwell_b200.kernels``."""
import math

import torch

own = False

HD = 128
EPS, BASE = 1e-6, 1e6
F8 = torch.float8_e4m3fn
EOS = 2


def listed():
    return [
        # one sequence's next token goes into the 8-bit cache: a launch and its latency
        {"name": "write-1", "kind": "write", "M": 1, "T": 1, "nq": 32, "nkv": 8, "at": 1500, "e4m3": True, "bf16": False, "tree": False},
        # portions of 512 prompt tokens of eight sequences: memory traffic
        {"name": "write-8x512", "kind": "write", "M": 8, "T": 512, "nq": 32, "nkv": 8, "at": 512, "e4m3": True, "bf16": False, "tree": False},
        # one user's next token over an 8-bit cache
        {"name": "decode-1", "kind": "attend", "M": 1, "T": 1, "nq": 32, "nkv": 8, "ctx": 2048, "e4m3": True, "bf16": False},
        # a server batch of unequal long contexts over an 8-bit cache
        {"name": "decode-32", "kind": "attend", "M": 32, "T": 1, "nq": 32, "nkv": 8, "ctx": 8192, "e4m3": True, "bf16": False},
        # small drafted trees, a group of seven query heads, the binary16 cache of the decode steps
        {"name": "tree-4x8", "kind": "attend", "M": 4, "T": 8, "nq": 28, "nkv": 4, "ctx": 1000, "e4m3": False, "bf16": False},
        # the widest trees on a server batch, bfloat16 activations: arithmetic outweighs the cache
        {"name": "tree-8x64", "kind": "attend", "M": 8, "T": 64, "nq": 32, "nkv": 8, "ctx": 4096, "e4m3": True, "bf16": True},
        # one request with four beams, a small vocabulary: latency
        {"name": "select-1x4", "kind": "select", "M": 1, "beams": 4, "vocab": 32768},
        # a batch of requests with eight beams over a large vocabulary of odd size: every logit is read
        {"name": "select-16x8", "kind": "select", "M": 16, "beams": 8, "vocab": 151643},
        # four beams a few tokens behind a prompt, six layers
        {"name": "reorder-1x4", "kind": "reorder", "M": 1, "beams": 4, "layers": 6, "nkv": 8, "start": 40, "rows": 61, "e4m3": True},
        # eight requests of four beams that share no prompt: a gigabyte of cache is rearranged
        {"name": "reorder-8x4", "kind": "reorder", "M": 8, "beams": 4, "layers": 6, "nkv": 8, "start": 0, "rows": 1500, "e4m3": False},
        # the accepted path of one small tree, all layers of a model
        {"name": "keep-1x8", "kind": "keep", "M": 1, "T": 8, "layers": 36, "nkv": 8, "first": 300, "e4m3": False},
        # accepted paths of the widest trees of a server batch
        {"name": "keep-32x64", "kind": "keep", "M": 32, "T": 64, "layers": 36, "nkv": 8, "first": 150, "e4m3": True},
    ]


HEADS = ((32, 8), (32, 8), (28, 4), (64, 8), (16, 16), (24, 8))


def _log(rng, lo, hi):
    hi = max(lo, int(hi))
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["write", "attend", "attend", "attend", "select", "select", "reorder", "keep"])
    case = {"kind": kind}
    if kind == "write":
        case["M"] = _log(rng, 1, 32)
        case["tree"] = rng.random() < 0.5
        case["nq"], case["nkv"] = rng.choice(HEADS)
        case["T"] = _log(rng, 1, min(64 if case["tree"] else 2048, 4096 * 32 / case["nq"] / case["M"]))
        case["at"] = _log(rng, 1, 30000 // case["M"])
        case["e4m3"], case["bf16"] = rng.random() < 0.7, rng.random() < 0.4
    elif kind == "attend":
        case["nq"], case["nkv"] = rng.choice(HEADS)
        case["M"] = _log(rng, 1, 32)
        case["T"] = 1 if rng.random() < 0.4 else rng.randint(2, 64)
        rows = min(32 * 8192 * 8 / (case["M"] * case["nkv"]), 8 * 64 * 4096 * 32 / (case["M"] * case["T"] * case["nq"]))
        case["ctx"] = _log(rng, 17, min(32768, rows))
        case["e4m3"], case["bf16"] = rng.random() < 0.6, rng.random() < 0.4
    elif kind == "select":
        case["beams"] = rng.randint(2, 16)
        case["vocab"] = _log(rng, 1000, 151643)
        case["M"] = _log(rng, 1, min(32, 16 * 8 * 151643 / (case["beams"] * case["vocab"])))
    elif kind == "reorder":
        case["M"], case["beams"] = _log(rng, 1, 8), rng.randint(2, 8)
        case["layers"], case["nkv"] = rng.randint(1, 6), rng.choice([4, 8, 16])
        case["e4m3"] = rng.random() < 0.5
        rows = 8 * 4 * 6 * 8 * 1500 / (case["M"] * case["beams"] * case["layers"] * case["nkv"])
        case["rows"] = _log(rng, 5, min(4000, rows))
        case["start"] = rng.randint(0, 100) if rng.random() < 0.5 and case["rows"] < 1000 else 0
    else:
        case["M"], case["T"] = _log(rng, 1, 32), rng.randint(3, 64)
        case["layers"], case["nkv"] = rng.randint(1, 36), rng.choice([4, 8])
        case["first"], case["e4m3"] = rng.randint(0, 150), rng.random() < 0.5
    return case


# ---------------------------------------------------------------------------------------------- sizes that the case alone gives
def _lengths(case):
    """Rows of each sequence before the nodes: between half of ctx and ctx."""
    return [case["ctx"] - int(case["ctx"] // 2 * (m * 0.618 % 1.0)) for m in range(case["M"])]


def _counts(case):
    """Nodes of each sequence: T, and fewer in every third one."""
    return [case["T"] if m % 3 != 2 else max(1, case["T"] * 2 // 3) for m in range(case["M"])]


def _accepted(case):
    return [2 + (5 * m + 3) % min(10, case["T"] - 2) if case["T"] > 2 else 1 for m in range(case["M"])]


def _row_bytes(case):
    return HD + 4 if case["e4m3"] else 2 * HD


def work(case):
    kind = case["kind"]
    if kind == "write":
        rows, e = case["M"] * case["T"], 2 if case["bf16"] else 4
        return {"bytes": rows * ((2 * case["nq"] + 2 * case["nkv"]) * HD * e + 2 * case["nkv"] * _row_bytes(case)),
                "flops": rows * (case["nq"] + case["nkv"]) * HD * 8}
    if kind == "attend":
        e = 2 if case["bf16"] else 4
        pairs = list(zip(_lengths(case), _counts(case)))
        return {"bytes": sum(2 * case["nkv"] * (n + c) * _row_bytes(case) + 2 * case["nq"] * c * HD * e for n, c in pairs),
                "flops": sum(4 * HD * case["nq"] * c * (n + min(c, 8) / 2) for n, c in pairs)}
    if kind == "select":
        n = case["M"] * case["beams"]
        return {"bytes": 4 * n * case["vocab"] + 24 * n, "flops": 4 * n * case["vocab"]}
    if kind == "reorder":
        moved = case["M"] * case["layers"] * 2 * case["nkv"] * case["rows"] * _row_bytes(case)
        return {"bytes": moved * (case["beams"] - 1 + case["beams"] // 2), "flops": 0}
    return {"bytes": 2 * sum(_accepted(case)) * case["layers"] * 2 * case["nkv"] * _row_bytes(case), "flops": 0}


# ---------------------------------------------------------------------------------------------- inputs
def _cache(g, shape, e4m3):
    """One side of a cache [M][layers][nkv][max_seq][128] and its scales."""
    x = torch.empty(shape + (HD,), dtype=torch.float16, device="cuda").normal_(generator=g)
    if not e4m3:
        return x, None
    scale = torch.empty(shape, device="cuda").uniform_(0.004, 0.012, generator=g)
    return (x * 110).clamp(-448, 448).to(F8), scale


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    s, kind = dict(case), case["kind"]

    def tree(M, T):
        """Parents of a random tree (each node's an earlier one, or none): depths [M, T] and ancestor masks [M, T], bit j: node j is seen."""
        u = torch.empty((M, T), device="cuda").uniform_(generator=g).cpu()
        depth, mask = torch.zeros((M, T), dtype=torch.int32), torch.zeros((M, T), dtype=torch.int64)
        for m in range(M):
            bits = [0] * T
            for i in range(T):
                p = int(u[m, i] * (i + 1)) - 1
                bits[i] = (bits[p] if p >= 0 else 0) | 1 << i
                depth[m, i] = depth[m, p] + 1 if p >= 0 else 0
            mask[m] = torch.tensor([b - (1 << 64) if b >> 63 else b for b in bits], dtype=torch.int64)
        return depth.cuda(), mask.cuda()

    if kind == "write":
        M, T, nq, nkv = case["M"], case["T"], case["nq"], case["nkv"]
        act = torch.bfloat16 if case["bf16"] else torch.float32
        s["max_seq"] = case["at"] + T + 8
        s["k"], s["ks"] = _cache(g, (M, 1, nkv, s["max_seq"]), case["e4m3"])
        s["v"], s["vs"] = _cache(g, (M, 1, nkv, s["max_seq"]), case["e4m3"])
        s["qkv"] = torch.empty((M * T, (nq + 2 * nkv) * HD), device="cuda").normal_(generator=g).to(act)
        s["qw"] = torch.empty(HD, device="cuda").uniform_(0.5, 1.5, generator=g)
        s["kw"] = torch.empty(HD, device="cuda").uniform_(0.5, 1.5, generator=g)
        s["first"] = _ints([case["at"] - (m * 37) % max(1, case["at"] // 2) for m in range(M)])
        s["offset"] = tree(M, T)[0] if case["tree"] else None
        s["q"] = torch.zeros((M * T, nq * HD), dtype=act, device="cuda")
    elif kind == "attend":
        M, T, nq, nkv = case["M"], case["T"], case["nq"], case["nkv"]
        act = torch.bfloat16 if case["bf16"] else torch.float32
        s["max_seq"] = case["ctx"] + T + 5
        s["k"], s["ks"] = _cache(g, (M, 1, nkv, s["max_seq"]), case["e4m3"])
        s["v"], s["vs"] = _cache(g, (M, 1, nkv, s["max_seq"]), case["e4m3"])
        s["q"] = (torch.empty((M * T, nq * HD), device="cuda").normal_(generator=g) * 1.5).to(act)
        s["first"], s["count"] = _ints(_lengths(case)), _ints(_counts(case))
        s["mask"] = tree(M, T)[1] if T > 1 else None
        s["out"] = torch.zeros((M * T, nq * HD), dtype=act, device="cuda")
    elif kind == "select":
        M, B, V = case["M"], case["beams"], case["vocab"]
        s["logits"] = torch.empty((M * B, V), device="cuda").normal_(generator=g) * 2.5
        s["score"] = -torch.empty((M, B), device="cuda").uniform_(5.0, 9.0, generator=g)
        s["ended"] = torch.empty((M, B), device="cuda").uniform_(generator=g) < 0.15
        s["parent"], s["token"] = _ints([[0] * B] * M), _ints([[0] * B] * M)
        s["score_out"], s["ended_out"] = torch.zeros((M, B), device="cuda"), torch.zeros((M, B), dtype=torch.bool, device="cuda")
    elif kind == "reorder":
        M, B, L, nkv = case["M"], case["beams"], case["layers"], case["nkv"]
        s["max_seq"] = case["start"] + case["rows"] + 20
        s["k"], s["ks"] = _cache(g, (M * B, L, nkv, s["max_seq"]), case["e4m3"])
        s["v"], s["vs"] = _cache(g, (M * B, L, nkv, s["max_seq"]), case["e4m3"])
        name = torch.empty((M, B), device="cuda").uniform_(generator=g).argsort(1)       # beam b of a fixed family is called name[b]
        s["parent"] = torch.zeros((M, B), dtype=torch.int32, device="cuda")
        s["parent"].scatter_(1, name, name[:, torch.arange(B, device="cuda") // 2].int())
        s["from"], s["to"] = _ints([case["start"]] * M), _ints([case["start"] + case["rows"]] * M)
    else:
        M, T, L, nkv = case["M"], case["T"], case["layers"], case["nkv"]
        s["max_seq"] = case["first"] + T + 20
        s["k"], s["ks"] = _cache(g, (M, L, nkv, s["max_seq"]), case["e4m3"])
        s["v"], s["vs"] = _cache(g, (M, L, nkv, s["max_seq"]), case["e4m3"])
        s["first"], s["count"] = _ints([case["first"] + m % 7 for m in range(M)]), _ints(_accepted(case))
        # an ascending choice of the nodes behind the first
        pick = torch.empty((M, T - 1), device="cuda").uniform_(generator=g).argsort(1)
        at = torch.arange(T, device="cuda").expand(M, T)
        pick = torch.where(at[:, :T - 1] < s["count"][:, None], pick + 1, T + at[:, :T - 1]).sort(1).values
        s["path"] = torch.cat([pick, at[:, :1] + 2 * T], 1).clamp(max=T - 1).int().contiguous()
    return s


# ---------------------------------------------------------------------------------------------- one pass
def run(s):
    if own:
        return _own(s)
    return {"write": _write, "attend": _attend, "select": _select, "reorder": _reorder, "keep": _keep}[s["kind"]](s)


def _with_scales(s, out):
    """The cache as it stands, after what the call returned."""
    return out + [s["k"], s["v"]] + ([s["ks"], s["vs"]] if s["e4m3"] else [])


def _bits(s):
    """The cache after a call that only moves rows, as the bits that it holds."""
    return [s["k"].view(torch.int16 if s["k"].dtype == torch.float16 else torch.int8), s["v"].view(torch.int16 if s["v"].dtype == torch.float16 else torch.int8)] + (
        [s["ks"].view(torch.int32), s["vs"].view(torch.int32)] if s["e4m3"] else [])


def _own(s):
    from blackwell_b200 import kernels as k

    kind = s["kind"]
    h = s.get("handle")
    if h is None:
        h = s["handle"] = {}
        if kind != "select":
            seqs, layers, nkv = s["k"].shape[:3]
            plane = nkv * s["max_seq"] * HD
            h["kv"] = k.KVCache(s["k"], s["v"], s["ks"], s["vs"], nkv, s["max_seq"], layers * plane, 0)
            h["plane"] = plane
        if kind == "attend":
            n = k.attention_tree_scratch_bytes(s["M"], s["T"], s["nq"], s["nkv"], s["max_seq"])
            h["scratch"] = torch.empty(n, dtype=torch.uint8, device="cuda")
        if kind == "select":
            n = k.beam_select_scratch_bytes(s["vocab"], s["beams"], s["beams"], s["M"])
            h["scratch"] = torch.empty(n, dtype=torch.uint8, device="cuda")
    if kind == "write":
        k.qk_norm_rope_kv_rows(s["q"], h["kv"], s["qkv"], s["qw"], s["kw"], s["first"], s["offset"], None, s["nq"], s["M"], s["T"], EPS, BASE)
        return _with_scales(s, [s["q"]])
    if kind == "attend":
        k.attention_tree(s["out"], s["q"], h["kv"], s["first"], s["mask"], s["count"], s["ctx"] + s["T"], s["nq"], s["M"], s["T"], h["scratch"])
        return s["out"]
    if kind == "select":
        k.beam_select(s["parent"], s["token"], s["score_out"], s["ended_out"], s["logits"], s["vocab"], s["vocab"], s["score"], s["ended"], EOS,
                      s["beams"], s["beams"], s["M"], h["scratch"])
        return [s["parent"], s["token"], s["score_out"], s["ended_out"]]
    if kind == "reorder":
        k.kv_reorder(h["kv"], s["parent"], s["from"], s["to"], s["beams"], s["M"], s["layers"], h["plane"])
        return _bits(s)
    k.kv_keep_rows(h["kv"], s["first"], s["path"], s["count"], s["M"], s["T"], s["layers"], h["plane"])
    return _bits(s)


def _write(s):
    M, T, nq, nkv = s["M"], s["T"], s["nq"], s["nkv"]
    x = s["qkv"].float().view(M, T, nq + 2 * nkv, HD)
    i = torch.arange(T, device="cuda")
    row = s["first"][:, None] + i
    pos = s["first"][:, None] + (i if s["offset"] is None else s["offset"])
    freq = torch.exp(torch.arange(HD // 2, device="cuda", dtype=torch.float64) * (-2 * math.log(BASE) / HD))
    angle = pos[..., None].double() * freq                      # far positions: 32 bits would lose the angle
    c, sn = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]

    def turned(y, w):
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w
        a, b = y[..., 0::2], y[..., 1::2]
        return torch.stack([a * c - b * sn, a * sn + b * c], -1).flatten(-2)

    s["q"].copy_(turned(x[:, :, :nq], s["qw"]).reshape(M * T, nq * HD))
    seq = torch.arange(M, device="cuda")[:, None]
    new = ((s["k"], s["ks"], turned(x[:, :, nq:nq + nkv], s["kw"])), (s["v"], s["vs"], x[:, :, nq + nkv:]))
    for side, scale, y in new:
        if s["e4m3"]:
            top = y.abs().amax(-1, keepdim=True)
            y = (y * (448.0 / top)).to(F8)
            scale[:, 0].transpose(1, 2)[seq, row] = top[..., 0] / 448.0
            side.view(torch.uint8)[:, 0].transpose(1, 2)[seq, row] = y.view(torch.uint8)
        else:
            side[:, 0].transpose(1, 2)[seq, row] = y.half()
    return _with_scales(s, [s["q"]])


def _attend(s):
    M, T, nq, nkv = s["M"], s["T"], s["nq"], s["nkv"]
    L = s["ctx"] + T
    kk, vv = s["k"][:, 0, :, :L].float(), s["v"][:, 0, :, :L].float()
    if s["e4m3"]:
        kk, vv = kk * s["ks"][:, 0, :, :L, None], vv * s["vs"][:, 0, :, :L, None]
    # queries [M, nkv, T * group, 128]
    q = s["q"].float().view(M, T, nkv, nq // nkv, HD).permute(0, 2, 1, 3, 4).reshape(M, nkv, -1, HD)
    at = torch.arange(L, device="cuda")
    node = at - s["first"][:, None]                              # [M, L]: which node lies in a row (negative: none)
    if s["mask"] is None:
        seen = (node[:, None] <= torch.arange(T, device="cuda")[:, None])
    else:
        bit = s["mask"][:, :, None] >> node.clamp(0, 63)[:, None] & 1
        seen = (node[:, None] < 0) | ((bit != 0) & (node < T)[:, None])
    score = q @ kk.transpose(-1, -2) * (1.0 / math.sqrt(HD))
    seen = seen[:, None, :, None].expand(M, nkv, T, nq // nkv, L).reshape(M, nkv, -1, L)
    score = torch.where(seen, score, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    o = p @ vv / p.sum(-1, keepdim=True)
    o = o.view(M, nkv, T, nq // nkv, HD).permute(0, 2, 1, 3, 4).reshape(M, T, nq * HD)
    live = torch.arange(T, device="cuda") < s["count"][:, None]
    return torch.where(live[..., None], o, 0.0).to(s["q"].dtype).view(M * T, nq * HD)


def _select(s):
    M, B, V = s["M"], s["beams"], s["vocab"]
    x = s["logits"].double().view(M, B, V)                       # candidates of two beams may lie next to each other
    top = x.amax(-1, keepdim=True)
    x = s["score"].double()[..., None] + (x - top - torch.log(torch.exp(x - top).sum(-1, keepdim=True)))
    only = torch.arange(V, device="cuda") == EOS
    x = torch.where(s["ended"][..., None], torch.where(only, s["score"].double()[..., None], -math.inf), x)
    best, at = x.view(M, B * V).topk(B, dim=1)                   # (normal logits: no two candidates are equal)
    parent, token = at // V, at % V
    return [parent.int(), token.int(), best.float(), s["ended"].gather(1, parent) | (token == EOS)]


def _reorder(s):
    M, B, lo, hi = s["M"], s["beams"], s["start"], s["start"] + s["rows"]
    src = (torch.arange(M, device="cuda")[:, None] * B + s["parent"]).view(-1)
    sides = [s["k"], s["v"]] + ([s["ks"], s["vs"]] if s["e4m3"] else [])
    for x in sides:
        x = x.view(torch.uint8) if x.dtype == F8 else x
        x[:, :, :, lo:hi] = x[src, :, :, lo:hi]
    return _bits(s)


def _keep(s):
    M, T = s["M"], s["T"]
    i = torch.arange(T, device="cuda")
    seq = torch.arange(M, device="cuda")[:, None]
    src = s["first"][:, None] + torch.where(i < s["count"][:, None], s["path"], i)
    dst = s["first"][:, None] + i
    sides = [s["k"], s["v"]] + ([s["ks"], s["vs"]] if s["e4m3"] else [])
    for x in sides:
        x = x.view(torch.uint8) if x.dtype == F8 else x
        x = x.transpose(1, 3)                                    # rows in front
        x[seq, dst] = x[seq, src]
    return _bits(s)


# ---------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    kind = case["kind"]
    if kind in ("reorder", "keep"):
        return None                                              # copies
    s = prepare(case, seed)
    M = case["M"]
    if kind == "select":
        B, V = case["beams"], case["vocab"]
        scores = torch.zeros((M, B), dtype=torch.float64)
        for m in range(M):
            rows = []
            for b in range(B):
                x, c = s["logits"][m * B + b].double(), float(s["score"][m, b])
                rows.append(torch.tensor([c], dtype=torch.float64, device="cuda") if s["ended"][m, b] else c + torch.log_softmax(x, 0))
            scores[m] = torch.cat(rows).sort(descending=True).values[:B].cpu()
        return [None, None, scores, None]
    T, nq, nkv = case["T"], case["nq"], case["nkv"]
    if kind == "write":
        half = torch.arange(0, HD, 2, device="cuda", dtype=torch.float64)
        heads = s["qkv"].double().view(M, T, -1, HD)
        q = torch.zeros((M, T, nq, HD), dtype=torch.float64, device="cuda")
        k, v = s["k"].double(), s["v"].double()
        ks, vs = (s["ks"].double(), s["vs"].double()) if case["e4m3"] else (None, None)
        first = s["first"].tolist()
        for m in range(M):
            step = s["offset"][m].double() if case["tree"] else torch.arange(T, device="cuda", dtype=torch.float64)
            turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), (first[m] + step)[:, None] * BASE ** (-half / HD))

            def norm_turn(x, w):
                x = x / (x.pow(2).sum(-1, keepdim=True) / HD + EPS).sqrt() * w.double()
                return torch.view_as_real(torch.view_as_complex(x.unflatten(-1, (HD // 2, 2)).contiguous()) * turn[:, None]).flatten(-2)

            q[m] = norm_turn(heads[m, :, :nq], s["qw"])
            for side, scale, x in ((k, ks, norm_turn(heads[m, :, nq:nq + nkv], s["kw"])), (v, vs, heads[m, :, nq + nkv:])):
                x = x.transpose(0, 1)
                if case["e4m3"]:                                 # (codes before their rounding to 8 bits)
                    unit = x.abs().max(-1).values / 448
                    scale[m, 0, :, first[m]:first[m] + T] = unit
                    x = x / unit[..., None]
                side[m, 0, :, first[m]:first[m] + T] = x
        return [q.view(M * T, nq * HD), k, v] + ([ks, vs] if case["e4m3"] else [])
    if M * T * nq * case["ctx"] > 1 << 29:
        return None
    group = nq // nkv
    out = torch.zeros((M, T, nq, HD), dtype=torch.float64, device="cuda")
    for m, (n, c) in enumerate(zip(_lengths(case), _counts(case))):
        k, v = s["k"][m, 0, :, :n + c].double(), s["v"][m, 0, :, :n + c].double()
        if case["e4m3"]:
            k, v = k * s["ks"][m, 0, :, :n + c, None].double(), v * s["vs"][m, 0, :, :n + c, None].double()
        q = s["q"].view(M, T, nq, HD)[m, :c].double()
        hide = torch.zeros((c, n + c), dtype=torch.bool)
        if T > 1:
            for i, bits in enumerate(s["mask"][m, :c].tolist()):
                hide[i, n:] = torch.tensor([not bits >> j & 1 for j in range(c)])
        for h in range(nq):
            logit = (q[:, h] @ k[h // group].T / HD ** 0.5).masked_fill(hide.cuda(), -math.inf)
            out[m, :c, h] = torch.softmax(logit, -1) @ v[h // group]
    return out.view(M * T, nq * HD)
