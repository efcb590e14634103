"""Workloads of the cached-attention operators: rope_append, paged_attention and kv_copy_pages.

Each case is one call of one operator with the tensors a decode program has in hand.  `run` computes it either in
plain torch operations (`own` false) or with this package's kernels (`own` true); `exact` computes the same outputs
from the formulas in 64 bits.  Head counts: 32 query / 8 key-value heads of 64 (Llama-3.2-1B), 24 / 8 of 128
(Llama-3.2-3B), and generic odd ones.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    attend = dict(op="attend", layout="heads", empty=0, shared=False)
    append = dict(op="append", layout="heads", interleaved=False, scaling="none", norm=False)
    copy = dict(op="copy", layout="heads")
    return [
        # the reference's chat prompt (53 tokens) in its own fp32 cache: the latency of one call
        dict(attend, name="attend one short", rows=1, lo=53, hi=53, kv_heads=8, group=4, dim=64, page=16, cache="f32"),
        # a small batch at the reference's default context limit, fp32 cache
        dict(attend, name="attend 16 fp32", rows=16, lo=1, hi=1024, kv_heads=8, group=4, dim=64, page=16, cache="f32"),
        # ordinary serving batch on the 1B model
        dict(attend, name="attend 16 bf16", rows=16, lo=1, hi=4096, kv_heads=8, group=4, dim=64, page=16, cache="bf16"),
        # one very long conversation on the 3B model: the split over the cache's length
        dict(attend, name="attend long", rows=1, lo=131072, hi=131072, kv_heads=8, group=3, dim=128, page=64,
             cache="bf16"),
        # a large ragged batch on the 3B model, some of its rows not in use
        dict(attend, name="attend 64 ragged", rows=64, lo=1, hi=8192, kv_heads=8, group=3, dim=128, page=16,
             cache="bf16", empty=3),
        # odd heads, head size, page size and lengths, token-major pages, rows that share sequences
        dict(attend, name="attend odd", rows=33, lo=1, hi=3001, kv_heads=5, group=7, dim=80, page=24, cache="f16",
             layout="tokens", shared=True),
        # one new token of the 1B model, fp32 cache: latency
        dict(append, name="append one", tokens=1, first=53, kv_heads=8, group=4, dim=64, rot=64, page=16, cache="f32",
             scaling="llama3"),
        # one decode step of a batch, with the norms of queries and keys
        dict(append, name="append 64 decode", tokens=64, first=4000, kv_heads=8, group=3, dim=128, rot=128, page=16,
             cache="bf16", scaling="llama3", norm=True),
        # a prompt chunk deep in a long context
        dict(append, name="append prompt", tokens=8192, first=122880, kv_heads=8, group=3, dim=128, rot=128, page=16,
             cache="bf16", scaling="llama3"),
        # interleaved pairs over part of an odd head, token-major pages, linear scaling
        dict(append, name="append odd", tokens=1999, first=7, kv_heads=5, group=7, dim=80, rot=36, page=24,
             cache="f16", layout="tokens", interleaved=True, scaling="linear", norm=True),
        # four sequences forked: the partly filled last page of each copied in all 16 layers of the 1B model
        dict(copy, name="copy fork", pairs=4, pages=64, layers=16, kv_heads=8, dim=64, page=16, cache="bf16"),
        # a cache compacted: 256 pages moved in all 28 layers of the 3B model
        dict(copy, name="copy compact", pairs=256, pages=700, layers=28, kv_heads=8, dim=128, page=16, cache="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    c = dict(op=rng.choice(["attend", "attend", "attend", "append", "append", "copy"]),
             layout=rng.choice(["heads", "tokens"]), cache=rng.choice(["f32", "f16", "bf16", "bf16"]),
             kv_heads=rng.choice([1, 2, 4, 5, 8, 8]), dim=rng.choice([64, 64, 80, 96, 128, 128, 256]),
             page=rng.choice([8, 16, 16, 24, 32, 64, 128]))
    token = c["kv_heads"] * c["dim"] * 2 * SIZES[c["cache"]]  # bytes of one token's keys and values
    if c["op"] == "attend":
        c.update(group=rng.choice([1, 2, 3, 4, 4, 5, 7, 8]), shared=rng.random() < 0.2)
        c["rows"] = _log(rng, 1, 256)
        # at most 1 GB of keys and values, and 0.5 M tokens of padded rows
        top = max(1, min(131072, (1 << 30) // (token * c["rows"]), (1 << 19) // c["rows"]))
        c["hi"] = _log(rng, 1, top)
        c["lo"] = rng.choice([1, c["hi"]])
        c["empty"] = rng.randint(0, c["rows"] // 8)
    elif c["op"] == "append":
        c.update(group=rng.choice([1, 2, 3, 4, 4, 5, 7, 8]), interleaved=rng.random() < 0.4,
                 scaling=rng.choice(["none", "linear", "llama3"]), norm=rng.random() < 0.5)
        c["rot"] = rng.choice([c["dim"], c["dim"], c["dim"] // 2, c["dim"] // 4, 36])
        c["tokens"] = _log(rng, 1, 4096)
        c["first"] = _log(rng, 1, 120000)
    else:
        c["layers"] = rng.choice([1, 2, 16, 28, 32])
        page = token * c["page"] * c["layers"]
        c["pairs"] = _log(rng, 1, max(1, min(256, (400 << 20) // page)))
        c["pages"] = 2 * c["pairs"] + rng.randint(1, 64)
    return c


def _lengths(case):
    """Tokens of every row: spread evenly over [lo, hi] in a mixed order, `empty` of them zero."""
    n, lo, hi = case["rows"], case["lo"], case["hi"]
    got = [hi if i == 0 else lo + int((hi - lo) * ((i * 0.6180339887498949) % 1.0)) for i in range(n)]
    for i in range(case["empty"]):
        got[n - 1 - i * max(1, n // (case["empty"] + 1))] = 0
    return got


def _cache(case, layers, pages, g):
    """Keys and values [layers, pages, kv_heads, page, dim], as views of pages that are laid out head by head or token
    by token."""
    h, p, d = case["kv_heads"], case["page"], case["dim"]
    shape = (layers, pages, h, p, d) if case["layout"] == "heads" else (layers, pages, p, h, d)
    k, v = (torch.empty(shape, dtype=DTYPES[case["cache"]], device="cuda").normal_(generator=g) for _ in range(2))
    return (k, v) if case["layout"] == "heads" else (k.transpose(2, 3), v.transpose(2, 3))


def _frequencies(case):
    """Radians per position of every pair: 500000^(-2i/rot); "linear": a quarter of it; "llama3": long wavelengths 32
    times longer, those between a quarter of 8192 and 8192 in part."""
    f = 500000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64, device="cuda") / case["rot"])
    if case["scaling"] == "linear":
        f = f / 4.0
    if case["scaling"] == "llama3":
        share = ((8192.0 * f / (2.0 * math.pi) - 1.0) / 3.0).clamp(0.0, 1.0)
        f = f * (share + (1.0 - share) / 32.0)
    return f


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def order(n):
        return torch.randperm(n, generator=g, device="cuda")

    s = {"case": case}
    if case["op"] == "copy":
        s["k"], s["v"] = _cache(case, case["layers"], case["pages"], g)
        mixed = order(case["pages"]).to(torch.int32)
        s["src"] = mixed[:case["pairs"]].contiguous()
        s["dst"] = mixed[case["pairs"]:2 * case["pairs"]].contiguous()
        return s
    h, d, p = case["kv_heads"], case["dim"], case["page"]
    heads = h * case["group"]
    if case["op"] == "attend":
        lengths = _lengths(case)
        rows = case["rows"]
        # where rows share sequences (several new tokens of one), two neighbours read the same pages
        s["seq"] = torch.arange(rows, device="cuda", dtype=torch.int32) // 2 if case["shared"] else None
        width = max(1, -(-max(lengths) // p))
        n = (rows + 1) // 2 if case["shared"] else rows
        s["k"], s["v"] = _cache(case, 1, n * width, g)
        s["table"] = order(n * width).to(torch.int32).reshape(n, width)
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        s["q"] = 2.0 * normal(rows, heads, d)  # scores with a standard deviation of 2: a few keys stand out
        s["out"] = torch.empty_like(s["q"])
        s["scale"] = d ** -0.5
        return s
    m = case["tokens"]
    # one sequence's prompt chunk; a batch's decode step has one token each
    decode = m <= 256
    n = m if decode else 1
    first = case["first"]
    spread = torch.arange(m, device="cuda")
    s["pos"] = ((first + spread * 37) % (first + 64) if decode else first + spread).to(torch.int32)
    s["seq"] = spread.to(torch.int32) if decode else torch.zeros(m, dtype=torch.int32, device="cuda")
    width = int(-(-(first + (64 if decode else m)) // p))
    # a page for every page that is written, the others' numbers wherever they come
    pages = n if decode else -(-m // p) + 1
    s["k_cache"], s["v_cache"] = _cache(case, 1, pages, g)
    if decode:
        s["table"] = order(pages).to(torch.int32)[:, None].expand(n, width).contiguous()
    else:
        s["table"] = torch.arange(width, device="cuda", dtype=torch.int32)[None] % pages
    s["q"], s["k"], s["v"] = normal(m, heads, d), normal(m, h, d), normal(m, h, d)
    s["q_out"] = torch.empty_like(s["q"])
    s["turns"] = _frequencies(case) / (2.0 * math.pi)  # turns per position
    s["q_norm"] = 1.0 + 0.1 * normal(d) if case["norm"] else None
    s["k_norm"] = 1.0 + 0.1 * normal(d) if case["norm"] else None
    return s


def _own(s):
    from minillama_infra_b200 import ops

    case = s["case"]
    if "cache" not in s:  # the handle that a program makes once for its cache
        k, v = (s["k_cache"], s["v_cache"]) if case["op"] == "append" else (s["k"], s["v"])
        s["cache"] = ops.KvCache(k, v)
        if case["op"] == "attend":
            s["workspace"] = ops.paged_attention_workspace(s["cache"], case["rows"], s["q"].shape[1])
    if case["op"] == "copy":
        ops.kv_copy_pages(s["cache"], s["src"], s["dst"])
        return {"k": s["k"], "v": s["v"]}
    if case["op"] == "attend":
        ops.paged_attention(s["out"], s["q"], s["cache"], 0, s["table"], s["lengths"], s["scale"], s["workspace"],
                            seq=s["seq"])
        return {"out": s["out"]}
    ops.rope_append(s["q_out"], s["q"], s["k"], s["v"], s["cache"], 0, s["pos"], s["table"], s["turns"], seq=s["seq"],
                    interleaved=case["interleaved"], q_norm=s["q_norm"], k_norm=s["k_norm"])
    return {"q": s["q_out"], "k": s["k_cache"], "v": s["v_cache"]}


def _rms(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w


def _rotate(x, cos, sin, interleaved):
    """Rotates the first 2 * cos.shape[-1] values of every head of x [m, heads, dim]."""
    half = cos.shape[-1]
    cos, sin = cos[:, None], sin[:, None]
    rot, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (rot[..., 0::2], rot[..., 1::2]) if interleaved else (rot[..., :half], rot[..., half:])
    y, z = a * cos - b * sin, b * cos + a * sin
    rot = torch.stack((y, z), -1).flatten(-2) if interleaved else torch.cat((y, z), -1)
    return torch.cat((rot, rest), -1)


def _plain_attend(s):
    case = s["case"]
    table = s["table"] if s["seq"] is None else s["table"][s["seq"].long()]
    rows, h, g, d = case["rows"], case["kv_heads"], case["group"], case["dim"]
    table = table.long()
    # [rows, kv_heads, tokens, dim]
    k, v = (x[0][table].permute(0, 2, 1, 3, 4).reshape(rows, h, -1, d).float() for x in (s["k"], s["v"]))
    far = torch.arange(k.shape[2], device="cuda") >= s["lengths"][:, None]
    scores = torch.matmul(s["q"].reshape(rows, h, g, d) * s["scale"], k.transpose(2, 3))
    scores = scores.masked_fill(far[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - top.masked_fill(top == -math.inf, 0.0))
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e, v) / total.masked_fill(total == 0.0, 1.0)
    s["out"].copy_(out.reshape(rows, h * g, d))
    return {"out": s["out"]}


def _plain_append(s):
    case = s["case"]
    angle = 2.0 * math.pi * torch.frac(s["pos"].double()[:, None] * s["turns"])
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    q, k = s["q"], s["k"]
    if case["norm"]:
        q, k = _rms(q, s["q_norm"]), _rms(k, s["k_norm"])
    s["q_out"].copy_(_rotate(q, cos, sin, case["interleaved"]))
    pos = s["pos"].long()
    page, slot = s["table"].long()[s["seq"].long(), pos // case["page"]], pos % case["page"]
    s["k_cache"][0][page, :, slot] = _rotate(k, cos, sin, case["interleaved"]).to(s["k_cache"].dtype)
    s["v_cache"][0][page, :, slot] = s["v"].to(s["v_cache"].dtype)
    return {"q": s["q_out"], "k": s["k_cache"], "v": s["v_cache"]}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "attend":
        return _plain_attend(state)
    if op == "append":
        return _plain_append(state)
    src, dst = state["src"].long(), state["dst"].long()
    state["k"][:, dst] = state["k"][:, src]
    state["v"][:, dst] = state["v"][:, src]
    return {"k": state["k"], "v": state["v"]}


def work(case):
    h, d, e = case["kv_heads"], case["dim"], SIZES[case["cache"]]
    if case["op"] == "copy":
        return {"bytes": 4.0 * case["pairs"] * case["layers"] * case["page"] * h * d * e, "flops": 0.0}
    heads = h * case["group"]
    if case["op"] == "attend":
        lengths = _lengths(case)
        read = [max(lengths[i:i + 2]) for i in range(0, len(lengths), 2)] if case["shared"] else lengths
        return {"bytes": 2.0 * sum(read) * h * d * e + 8.0 * case["rows"] * heads * d,
                "flops": 4.0 * sum(lengths) * heads * d}
    m = case["tokens"]
    return {"bytes": m * d * (8.0 * heads + 8.0 * h + 2.0 * e * h),
            "flops": m * (3.0 * (heads + h) * case["rot"] + (4.0 * (heads + h) * d if case["norm"] else 0.0))}


def exact(case, seed):
    if case["op"] == "copy":
        return None
    s = prepare(case, seed)
    h, g, d, p = case["kv_heads"], case["group"], case["dim"], case["page"]
    if case["op"] == "attend":
        out = torch.zeros(case["rows"], h * g, d, dtype=torch.float64, device="cuda")
        for r, n in enumerate(_lengths(case)):
            if n == 0:
                continue
            pages = s["table"][r // 2 if case["shared"] else r][:-(-n // p)].long()
            for j in range(h):
                k, v = (x[0, pages, j].reshape(-1, d)[:n].double() for x in (s["k"], s["v"]))
                weight = torch.softmax(s["q"][r, j * g:(j + 1) * g].double() @ k.T / math.sqrt(d), -1)
                out[r, j * g:(j + 1) * g] = weight @ v
        return {"out": out}
    m, rot = case["tokens"], case["rot"]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["pos"].double()[:, None] * _frequencies(case))

    def place(x, w):
        x = x.double()
        if w is not None:
            x = x * w.double() / torch.sqrt(x.square().sum(-1, keepdim=True) / d + 1e-5)
        at = torch.arange(rot // 2, device="cuda")
        i, j = (2 * at, 2 * at + 1) if case["interleaved"] else (at, at + rot // 2)
        z = torch.complex(x[..., i], x[..., j]) * turn[:, None]
        x = x.clone()
        x[..., i], x[..., j] = z.real, z.imag
        return x

    q, k = place(s["q"], s["q_norm"]), place(s["k"], s["k_norm"])
    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    seq, pos = s["seq"].long(), s["pos"].long()
    page = s["table"].long()[seq, torch.div(pos, p, rounding_mode="floor")]
    for j in range(h):
        k_cache[0, page, j, pos % p] = k[:, j]
        v_cache[0, page, j, pos % p] = s["v"][:, j].double()
    return {"q": q, "k": k_cache, "v": v_cache}
