"""What the 8-bit serving operators are measured on: the inputs, the plain forms, the calls.

Four operators that a layer runs one after the other: quantising activation rows, the 8-bit
integer product with token and channel scales, appending to an 8-bit paged cache (norm and
rotation on the way), and attention over that cache. `run` computes them in elementary torch
operations, or, where `own` is true, with the framework's kernels.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ESIZE = {"f32": 4, "f16": 2, "bf16": 2}
TINY = 2.0 ** -100  # groups whose largest magnitude is below this hold zeros
EPS = 1e-6


def listed():
    return [
        # one decoded token's layer input before its product
        dict(name="quantize_token", op="quantize", rows=1, cols=4096, type="f32"),
        # the down projection's input of a long prompt
        dict(name="quantize_prompt", op="quantize", rows=8192, cols=12288, type="bf16"),
        # the fused q, k, v product of one decoded token (4096 + 2 x 1024 rows)
        dict(name="matmul_token", op="matmul", rows=1, out=6144, cols=4096, type="f32", add=False),
        # the down projection of a batch of 33 sequences, 32B shape, into the residual
        dict(name="matmul_batch", op="matmul", rows=33, out=5120, cols=25600, type="bf16", add=True),
        # gate and up of a prompt, 8B shape
        dict(name="matmul_prompt", op="matmul", rows=4096, out=24576, cols=4096, type="bf16", add=False),
        # a decode step of 32 sequences writes its tokens, q and k normed
        dict(name="append_step", op="append", seqs=32, tokens=1, context=2048, heads=32, kv_heads=8, dim=128,
             rope=128, interleaved=False, norm=True, page=16, type="bf16"),
        # four prompts of uneven lengths enter the cache behind short prefixes, partial rotation, wide heads
        dict(name="append_prompt", op="append", seqs=4, tokens=5003, context=300, heads=16, kv_heads=4, dim=256,
             rope=64, interleaved=True, norm=False, page=64, type="f16"),
        # one sequence decodes at a short context
        dict(name="attend_short", op="attend", seqs=1, tokens=1, context=517, heads=32, kv_heads=8, dim=128,
             page=16, type="f32"),
        # a decode step of 32 sequences around 2048 positions
        dict(name="attend_step", op="attend", seqs=32, tokens=1, context=2100, heads=32, kv_heads=8, dim=128,
             page=16, type="bf16"),
        # one sequence decodes at a very long context
        dict(name="attend_long", op="attend", seqs=1, tokens=1, context=131071, heads=32, kv_heads=8, dim=128,
             page=64, type="f32"),
        # drafted tokens checked together: 4 new ones for each of 9 sequences, wide heads
        dict(name="attend_drafts", op="attend", seqs=9, tokens=4, context=4099, heads=16, kv_heads=2, dim=256,
             page=32, type="f16"),
        # a prompt's chunk attends to itself and to what came before it
        dict(name="attend_prompt", op="attend", seqs=1, tokens=2048, context=8192, heads=32, kv_heads=8, dim=128,
             page=16, type="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "matmul", "append", "attend"])
    kind = rng.choice(["f32", "f16", "bf16"])
    if op == "quantize":
        rows = _log(rng, 1, 8192)
        return dict(op=op, rows=rows, cols=_log(rng, 64, min(16384, 8192 * 12288 // rows)), type=kind)
    if op == "matmul":
        rows, out = _log(rng, 1, 4096), _log(rng, 64, 24576)
        return dict(op=op, rows=rows, out=out, cols=_log(rng, 64, 25600 if rows < 512 else 4096), type=kind,
                    add=rng.random() < 0.5)
    dim, group, kv_heads = rng.choice([64, 128, 256]), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 8])
    shape = dict(heads=group * kv_heads, kv_heads=kv_heads, dim=dim, page=rng.choice([16, 32, 64]), type=kind)
    if op == "append":
        seqs, most = _log(rng, 1, 64), min(20000, 120_000_000 // (shape["heads"] * dim * ESIZE[kind]))
        return dict(op=op, seqs=seqs, tokens=_log(rng, 1, max(1, most // seqs)), context=_log(rng, 1, 4096), **shape,
                    rope=rng.choice([0, dim // 4, dim // 2, dim]), interleaved=rng.random() < 0.3,
                    norm=rng.random() < 0.5)
    seqs = _log(rng, 1, 48)
    tokens = rng.choice([1, 1, 1, rng.randint(2, 16), _log(rng, 17, min(1024, 4_000_000 // (shape["heads"] * dim)))])
    if tokens > 16:
        seqs = min(seqs, 3)
    return dict(op=op, seqs=seqs, tokens=tokens,
                context=tokens + _log(rng, 1, 65000 // seqs if tokens <= 16 else 4096), **shape)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _activations(g, shape, kind):
    """Normal values with a few channels that are many times larger, as layer inputs have."""
    x = torch.randn(shape, generator=g, device=DEV)
    loud = torch.rand(shape[-1], generator=g, device=DEV) < 0.01
    return (x * torch.where(loud, 8.0, 1.0)).to(TYPES[kind])


def _spread(n, top, least):
    """n whole numbers in [least, top], the first of them `top`: a case's uneven lengths, known to host and device."""
    g = torch.Generator().manual_seed(77 + top)
    v = (top * (0.5 + 0.5 * torch.rand(n, generator=g))).long().clamp(min=least)
    v[0] = top
    return v.tolist()


def _cache(g, c, lens, room=0):
    """Pages in scattered order with codes and scales such as appended blocks have."""
    page, hk, dim = c["page"], c["kv_heads"], c["dim"]
    need = [-(-(n + room) // page) for n in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=DEV).int()
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    codes = [torch.randn((pages, hk, page, dim), generator=g, device=DEV).mul_(40).round_().clamp_(-127, 127).to(torch.int8)
             for _ in range(2)]
    scales = [torch.exp(torch.randn((pages, hk, page // 16), generator=g, device=DEV) * 0.3) / 40 for _ in range(2)]
    return {"k": codes[0], "v": codes[1], "ks": scales[0], "vs": scales[1], "table": table}


def _batch(c):
    """Lengths (after the new tokens) and new tokens of each sequence, on the host and on the device."""
    new, lens = _spread(c["seqs"], c["tokens"], 1), _spread(c["seqs"], c["context"], 0)
    lens = [a + b if c["op"] == "append" else max(a, b) for a, b in zip(lens, new)]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return {"new": new, "lens": lens, "cu": torch.tensor(cu, dtype=torch.int32, device=DEV),
            "len": torch.tensor(lens, dtype=torch.int32, device=DEV), "total": cu[-1], "max_q": max(new),
            "max_kv": max(lens)}


def prepare(case, seed):
    c, g = case, _gen(seed)
    if c["op"] == "quantize":
        return {"c": c, "x": _activations(g, (c["rows"], c["cols"]), c["type"]),
                "codes": torch.empty((c["rows"], -(-c["cols"] // 16) * 16), dtype=torch.int8, device=DEV)[:, :c["cols"]],
                "scales": torch.empty(c["rows"], device=DEV)}
    if c["op"] == "matmul":
        wide = -(-c["cols"] // 16) * 16  # rows of codes start on 16-byte boundaries
        s = {"c": c}
        for name, rows in (("x", c["rows"]), ("w", c["out"])):
            codes = torch.randn((rows, wide), generator=g, device=DEV).mul_(36).round_().clamp_(-127, 127).to(torch.int8)
            s[name] = codes[:, :c["cols"]]
            s[name + "s"] = (0.5 + torch.rand(rows, generator=g, device=DEV)) * (0.03 if name == "x" else 0.0006)
        s["add"] = torch.randn((c["rows"], c["out"]), generator=g, device=DEV).to(TYPES[c["type"]]) if c["add"] else None
        s["y"] = torch.empty((c["rows"], c["out"]), dtype=TYPES[c["type"]], device=DEV)
        return s
    b = _batch(c)
    s = {"c": c, **b, **_cache(g, c, b["lens"])}
    heads, hk, dim, kind = c["heads"], c["kv_heads"], c["dim"], c["type"]
    if c["op"] == "attend":
        s["q"] = (torch.randn((b["total"], heads, dim), generator=g, device=DEV) * 1.5).to(TYPES[kind])
        s["out"] = torch.empty_like(s["q"])
        return s
    # q, k and v are slices of one product's output, as a layer has them
    qkv = _activations(g, (b["total"], (heads + 2 * hk) * dim), kind)
    s["q"] = qkv[:, :heads * dim].unflatten(1, (heads, dim))
    s["kn"] = qkv[:, heads * dim:(heads + hk) * dim].unflatten(1, (hk, dim))
    s["vn"] = qkv[:, (heads + hk) * dim:].unflatten(1, (hk, dim))
    s["q_out"] = torch.empty((b["total"], heads, dim), dtype=TYPES[kind], device=DEV)
    s["rope"] = None
    if c["rope"]:
        i = torch.arange(c["rope"] // 2, device=DEV, dtype=torch.float64)
        angle = torch.outer(torch.arange(b["max_kv"], device=DEV, dtype=torch.float64), 1e6 ** (-2 * i / c["rope"]))
        s["rope"] = torch.stack([angle.cos(), angle.sin()], -1).float()
    s["q_norm"] = s["k_norm"] = None
    if c["norm"]:
        s["q_norm"], s["k_norm"] = (1 + 0.1 * torch.randn(dim, generator=g, device=DEV) for _ in range(2))
    # blocks that the new tokens touch, which the host knows from the lengths
    s["blocks"] = sum((n - 1) // 16 - (n - m) // 16 + 1 for n, m in zip(b["lens"], b["new"]))
    return s


# ------------------------------------------------------------------ the plain forms
def _scale_of(amax):
    s = amax / torch.full_like(amax, 127.0)
    s = torch.where(amax < TINY, torch.zeros_like(s), s)
    return torch.where(torch.isfinite(amax), s, torch.full_like(s, math.nan))


def _codes_of(x, scale):
    inv = torch.where(scale > 0, torch.reciprocal(scale), torch.zeros_like(scale))
    return torch.round(x * inv).nan_to_num(0.0).clamp(-127, 127).to(torch.int8)


def _plain_quantize(s):
    x = s["x"].float()
    scale = _scale_of(x.abs().amax(1))
    return {"codes": _codes_of(x, scale[:, None]), "scales": scale}


def _plain_matmul(s):
    y = s["x"].float() @ s["w"].float().T
    y = y * s["xs"][:, None] * s["ws"]
    if s["add"] is not None:
        y = y + s["add"].float()
    return {"y": y.to(s["y"].dtype)}


def _tokens(s):
    """The sequence, the place among the new ones and the position of each new token."""
    t = torch.arange(s["total"], device=DEV)
    seq = torch.searchsorted(s["cu"][1:].long(), t, right=True)
    i = t - s["cu"][seq]
    return seq, i, s["len"][seq] - (s["cu"][seq + 1] - s["cu"][seq]) + i


def _turn(x, norm, rope, pos, interleaved):
    """RMS norm (its sum in 64 bits) and the rotation by the table's rows."""
    x = x.float()
    if norm is not None:
        ms = x.double().square().mean(-1, keepdim=True)
        x = x * (1.0 / torch.sqrt(ms + EPS)).float() * norm
    if rope is None:
        return x
    half = rope.shape[1]
    cos, sin = rope[pos, :, 0][:, None], rope[pos, :, 1][:, None]
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    y, z = a * cos - b * sin, a * sin + b * cos
    r = torch.stack([y, z], -1).flatten(-2) if interleaved else torch.cat([y, z], -1)
    return torch.cat([r, x[..., 2 * half:]], -1)


def _plain_block_write(x, codes, scales, page, block, row, lead):
    """New rows x [T][kv heads][dim] into their blocks: the scale grows, older rows follow it."""
    n, hk, ps, dim = codes.shape
    per = ps // 16
    flat = (page * per + block).long()
    amax = torch.zeros((n * per, hk), device=DEV).index_reduce_(0, flat, x.abs().amax(-1), "amax")
    lp, lb, lr = page[lead].long(), block[lead].long(), row[lead]
    lf = flat[lead]
    old = torch.where((lr == 0)[:, None], 0.0, scales[lp, :, lb])
    new = torch.maximum(old, _scale_of(amax[lf]))
    ratio = torch.where(new > 0, old / new, torch.zeros_like(new))
    cells = codes.view(n, hk, per, 16, dim)
    was = cells[lp, :, lb]
    moved = torch.round(was.float() * ratio[..., None, None]).to(torch.int8)
    earlier = torch.arange(16, device=DEV)[None, None, :, None] < lr[:, None, None, None]
    cells[lp, :, lb] = torch.where(earlier, moved, was)
    scales[lp, :, lb] = new
    cells[page.long(), :, block.long(), row.long()] = _codes_of(x, scales[page.long(), :, block.long()][..., None])


def _plain_append(s):
    c = s["c"]
    seq, i, pos = _tokens(s)
    page = s["table"][seq, pos // c["page"]]
    block, row = pos % c["page"] // 16, pos % 16
    first = (i == 0) | (row == 0)
    lead = torch.argsort((~first).to(torch.int8), stable=True)[:s["blocks"]]
    k = _turn(s["kn"], s["k_norm"], s["rope"], pos, c["interleaved"])
    _plain_block_write(k, s["k"], s["ks"], page, block, row, lead)
    _plain_block_write(s["vn"].float(), s["v"], s["vs"], page, block, row, lead)
    q = _turn(s["q"], s["q_norm"], s["rope"], pos, c["interleaved"]).to(s["q_out"].dtype)
    # the whole cache, as the codes and the scales that it holds: equal codes, not near values
    return {"q": q, "k": s["k"], "v": s["v"], "ks": s["ks"], "vs": s["vs"]}


def _values(codes, scales, table, max_kv):
    """[sequences][kv heads][positions][dim] in 32 bits."""
    n, hk, ps, dim = codes.shape
    at = table[:, :-(-max_kv // ps)].clamp(min=0).long()
    x = codes[at].float().unflatten(3, (ps // 16, 16)) * scales[at][..., None, None]
    return x.flatten(3, 4).transpose(1, 2).flatten(2, 3)[:, :, :max_kv]


def _plain_attend(s):
    c = s["c"]
    n, hk, dim, group = c["seqs"], c["kv_heads"], c["dim"], c["heads"] // c["kv_heads"]
    seq, i, pos = _tokens(s)
    k, v = (_values(s[a], s[b], s["table"], s["max_kv"]) for a, b in (("k", "ks"), ("v", "vs")))
    q = torch.zeros((n, s["max_q"], hk, group, dim), device=DEV)
    q[seq, i] = s["q"].float().unflatten(1, (hk, group))
    limit = torch.full((n, s["max_q"]), -1, device=DEV)
    limit[seq, i] = pos
    q = q.permute(0, 2, 3, 1, 4).flatten(2, 3)
    x = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(dim))
    hide = torch.arange(s["max_kv"], device=DEV) > limit[:, None, None, :, None]
    x = x.unflatten(2, (group, s["max_q"])).masked_fill(hide, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
    total = x.sum(-1, keepdim=True)
    x = (x / torch.where(total > 0, total, torch.ones_like(total))).flatten(2, 3)
    o = (x @ v).unflatten(2, (group, s["max_q"])).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return {"out": o[seq, i].to(s["out"].dtype)}


PLAIN = {"quantize": _plain_quantize, "matmul": _plain_matmul, "append": _plain_append, "attend": _plain_attend}


# ------------------------------------------------------------------ the framework's calls
def _own(s):
    from evelyn_b200 import int8

    c = s["c"]
    if c["op"] == "quantize":
        int8.quantize_rows(s["x"], s["codes"], s["scales"])
        return {"codes": s["codes"], "scales": s["scales"]}
    if c["op"] == "matmul":
        int8.matmul(s["x"], s["xs"], s["w"], s["ws"], s["y"], add=s["add"])
        return {"y": s["y"]}
    if "kv" not in s:  # a server describes its pages and its batch's buffers once
        s["kv"] = int8.Kv8Cache(s["k"], s["v"], s["ks"], s["vs"])
        s["batch"] = int8.Kv8Batch(s["table"], s["cu"], s["len"], s["max_q"], s["max_kv"])
    cache, batch = s["kv"], s["batch"]
    if c["op"] == "append":
        int8.kv8_append(cache, batch, s["kn"], s["vn"], q=s["q"], q_out=s["q_out"], rope=s["rope"],
                        interleaved=c["interleaved"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
        return {"q": s["q_out"], "k": s["k"], "v": s["v"], "ks": s["ks"], "vs": s["vs"]}
    if "ws" not in s:  # a server keeps its workspace
        s["ws"] = torch.empty(int8.kv8_attention_workspace(cache, batch, s["q"]), dtype=torch.uint8, device=DEV)
    int8.kv8_attention(cache, batch, s["q"], s["out"], workspace=s["ws"])
    return {"out": s["out"]}


def run(state):
    return _own(state) if own else PLAIN[state["c"]["op"]](state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c, e = case, ESIZE[case["type"]]
    if c["op"] == "quantize":
        n = c["rows"] * c["cols"]
        return {"bytes": n * (e + 1) + 4 * c["rows"], "flops": 2 * n}
    if c["op"] == "matmul":
        m, n, k = c["rows"], c["out"], c["cols"]
        return {"bytes": (m + n) * (k + 4) + m * n * e * (2 if c["add"] else 1), "flops": 2 * m * n * k}
    new = 0.75 * c["tokens"] * c["seqs"] if c["seqs"] > 1 and c["tokens"] > 1 else c["tokens"] * c["seqs"]
    heads, hk, dim = c["heads"], c["kv_heads"], c["dim"]
    if c["op"] == "append":
        per = (2 * heads + 2 * hk) * dim * e + 2 * hk * dim + 2 * hk * 4 / 16 + 4 * c["rope"]
        return {"bytes": new * per, "flops": new * (heads + 2 * hk) * dim * 8}
    kv = c["context"] * (0.75 * c["seqs"] if c["seqs"] > 1 else 1)
    seen = kv - (c["tokens"] - 1) / 2 * (0.75 * c["seqs"] if c["seqs"] > 1 else 1)
    return {"bytes": kv * 2 * hk * (dim + 0.25) + 2 * new * heads * dim * e,
            "flops": 4 * heads * dim * seen * new / c["seqs"]}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_turn(x, norm, rope, pos, interleaved):
    x = x.double()
    if norm is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * norm.double()
    if rope is None:
        return x
    half = rope.shape[1]
    turn = torch.complex(rope[pos, :, 0].double(), rope[pos, :, 1].double())[:, None]
    head = x[..., :2 * half]
    pairs = head.unflatten(-1, (half, 2)) if interleaved else head.unflatten(-1, (2, half)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    x = x.clone()
    x[..., :2 * half] = z.flatten(-2) if interleaved else z.transpose(-1, -2).flatten(-2)
    return x


def _exact_scales(x, scales, s, page):
    """Block scales after the new rows x [T][kv heads][dim], sequence by sequence."""
    scales, table, at = scales.double(), s["table"].tolist(), 0
    for q, (n, m) in enumerate(zip(s["lens"], s["new"])):
        p = n - m
        while p < n:
            end = min(n, p // 16 * 16 + 16)
            top = x[at:at + end - p].abs().amax((0, 2)) / 127
            cell = scales[table[q][p // page], :, p % page // 16]
            cell.copy_(top if p % 16 == 0 else torch.maximum(cell, top))
            at, p = at + end - p, end
    return scales


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "quantize":
        return {"codes": None, "scales": s["x"].double().abs().amax(1) / 127}
    if c["op"] == "matmul":
        y = torch.matmul(s["x"].double(), s["w"].double().T) * torch.outer(s["xs"].double(), s["ws"].double())
        return {"y": y if s["add"] is None else y + s["add"].double()}
    seqs = torch.repeat_interleave(torch.arange(c["seqs"]), torch.tensor(s["new"]))
    pos = torch.cat([torch.arange(n - m, n) for n, m in zip(s["lens"], s["new"])]).to(DEV)
    if c["op"] == "append":
        k = _exact_turn(s["kn"], s["k_norm"], s["rope"], pos, c["interleaved"])
        return {"q": _exact_turn(s["q"], s["q_norm"], s["rope"], pos, c["interleaved"]), "k": None, "v": None,
                "ks": _exact_scales(k, s["ks"], s, c["page"]),
                "vs": _exact_scales(s["vn"].double(), s["vs"], s, c["page"])}
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    group, at, ps = c["heads"] // c["kv_heads"], 0, c["page"]
    for b, (n, m) in enumerate(zip(s["lens"], s["new"])):
        pages = s["table"][b, :-(-n // ps)].long()
        kv = []
        for codes, scales in ((s["k"], s["ks"]), (s["v"], s["vs"])):
            x = codes[pages].double() * scales[pages].double().repeat_interleave(16, 2)[..., None]
            kv.append(x.transpose(0, 1).reshape(c["kv_heads"], -1, c["dim"])[:, :n])
        for t in range(0, m, 256):  # rows at a time, to bound the scores in memory
            e = min(m, t + 256)
            q = s["q"][at + t:at + e].double()
            here = torch.arange(n - m + t, n - m + e, device=DEV)
            for h in range(c["heads"]):
                x = q[:, h] @ kv[0][h // group].T / math.sqrt(c["dim"])
                x = x.masked_fill(torch.arange(n, device=DEV)[None] > here[:, None], -math.inf)
                out[at + t:at + e, h] = torch.softmax(x, -1) @ kv[1][h // group]
        at += m
    return {"out": out}
