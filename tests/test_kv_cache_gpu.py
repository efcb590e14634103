"""The cached-attention operators on the GPU against their formulas in 64 bits.

Tolerances count roundings of u = 2^-24 (fp32) and of half a step of the cache's
type:
  * rope_append: a norm's factor carries the roundings of a sum of squares
    (at most 8 terms a lane and 5 levels), a quotient and a root, a weight; an
    angle is off by pi 2^-24 after its rounding to fp32 and its sine and cosine
    by 2 units; a rotated value is two products and a sum.  All of it stays
    below 32 u (|a| + |b|) for the pair (a, b).
  * paged_attention: a score s = scale q.k is a sum of head_dim products taken
    as at most head_dim / 4 + 16 steps that each lose at most u of
    S = scale sum |q k|; it is off by ds = (head_dim / 4 + 16) u S.  Weights
    and their sum then are off by 2 ds, by the argument's and the result's roundings
    (2 S + 4) u, and the sums over tokens by 32 u within a tile and, for n tokens,
    8 sqrt(n) u over all: independent roundings add as their root.  The output is off
    by at most all of that times A = sum p |v| (bound per value), and, in the
    root mean square over a row, where the score's roundings are independent
    too, by (8 sqrt(head_dim) + 8 sqrt(n) + 16) u A.
  * copies and values (v): equal.
"""
import math

import numpy as np
import pytest

from minillama_infra_b200 import ops
from minillama_infra_b200._lib import MliError
from minillama_infra_b200.kv_cache import PagedKvCache

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
GUARD = 64


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def empty_cache(layers, pages, heads, page, dim, dtype, layout="heads", fill=math.nan):
    inner = (heads, page) if layout == "heads" else (page, heads)
    k, v = (torch.full((layers, pages, *inner, dim), fill, dtype=dtype, device="cuda") for _ in range(2))
    return ops.KvCache(*((k, v) if layout == "heads" else (k.transpose(2, 3), v.transpose(2, 3))))


def guarded(rows, width):
    """A float matrix [rows, width] between two bands of NaN, and a check of the bands."""
    buf = torch.full((rows * width + 2 * GUARD,), math.nan, device="cuda")

    def check():
        assert buf[:GUARD].isnan().all() and buf[-GUARD:].isnan().all(), "guard band overwritten"

    return buf[GUARD:GUARD + rows * width].view(rows, width), check


def filled(g, lengths, heads, page, dim, dtype, layout="heads", layers=1, layer=0, spare=3):
    """A cache whose pages hold the sequences' keys and values in a mixed order and NaN everywhere else."""
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + spare
    c = empty_cache(layers, pages, heads, page, dim, dtype, layout)
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    table = np.full((len(lengths), max(1, max(counts))), -1, np.int32)
    kv = []
    for s, n in enumerate(lengths):
        k, v = (normal(g, n, heads, dim).to(dtype) for _ in range(2))
        kv.append((k, v))
        for j in range(counts[s]):
            table[s, j] = p = order.pop()
            m = min(page, n - j * page)
            c.k[layer, p, :, :m] = k[j * page:j * page + m].transpose(0, 1)
            c.v[layer, p, :, :m] = v[j * page:j * page + m].transpose(0, 1)
    return c, torch.from_numpy(table).cuda(), kv


def attention64(q, k, v, scale):
    """(out, A, S) of one row in 64 bits: q [heads, dim], k, v [n, kv_heads, dim]."""
    group = q.shape[0] // k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    k, v = (x.transpose(0, 1).repeat_interleave(group, 0) for x in (k, v))  # [heads, n, dim]
    s = scale * (k @ q[..., None]).squeeze(-1)
    p = torch.softmax(s, -1)[:, None]
    size = scale * (k.abs() @ q.abs()[..., None]).amax((1, 2))
    return (p @ v).squeeze(1), (p @ v.abs()).squeeze(1), size


def check_row(got, q, k, v, scale, what=""):
    n, dim = k.shape[0], q.shape[1]
    if n == 0:
        assert (got == 0).all(), what
        return
    want, a, size = attention64(q, k, v, scale)
    err = (got.double() - want).abs()
    size = size[:, None]
    bound = (2 * (dim / 4 + 16) * size + 2 * size + 4 + 32 + 8 * math.sqrt(n)) * U * a
    assert torch.isfinite(got).all() and (err <= bound).all(), (what, (err / bound).max())
    rms = (8 * math.sqrt(dim) + 8 * math.sqrt(n) + 16) * U * a.square().mean(-1).sqrt()
    assert (err.square().mean(-1).sqrt() <= rms).all(), (what, (err.square().mean(-1).sqrt() / rms).max())


def attend(c, table, q, lengths, scale, seq=None, layer=0, ws=None):
    """paged_attention into guarded memory, twice: the same bits."""
    rows, heads, dim = q.shape
    ws = ops.paged_attention_workspace(c, rows, heads) if ws is None else ws
    got = []
    for _ in range(2):
        out, check = guarded(rows, heads * dim)
        ops.paged_attention(out.view(rows, heads, dim), q, c, layer, table, lengths, scale, ws, seq=seq)
        torch.cuda.synchronize()
        check()
        got.append(out.view(rows, heads, dim).clone())
    assert torch.equal(got[0].view(torch.int32), got[1].view(torch.int32))
    return got[0]


# lengths, kv_heads, group, dim, page
ATTENTION = [
    ([1], 1, 1, 64, 16), ([53], 8, 4, 64, 16), ([0, 1, 2, 15, 16, 17, 31, 32, 33, 0], 2, 4, 64, 16),
    ([5000, 3, 0, 700], 8, 4, 64, 16), ([1000, 999], 8, 3, 128, 16), ([65, 64, 63, 127, 128, 129, 130], 4, 8, 128, 32),
    ([300, 7], 2, 16, 128, 8), ([90, 1000], 1, 9, 64, 16), ([257, 1], 5, 7, 80, 24), ([100, 200, 300], 3, 5, 96, 1),
    ([2000, 31], 2, 2, 256, 16), ([100, 9], 2, 8, 256, 64), ([77, 5], 1, 2, 8, 16), ([400], 4, 1, 128, 128),
    ([33000], 2, 4, 64, 64), ([70000], 1, 1, 64, 7), (list(range(0, 300)), 1, 4, 64, 16), ([40] * 200, 4, 6, 64, 16),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", range(len(ATTENTION)))
def test_attention(case, dtype):
    lengths, heads, group, dim, page = ATTENTION[case]
    g = gen(100 + case)
    c, table, kv = filled(g, lengths, heads, page, dim, dtype, "heads" if case % 2 else "tokens", layers=2, layer=1)
    q = normal(g, len(lengths), heads * group, dim)
    scale = dim ** -0.5
    got = attend(c, table, q, i32(lengths), scale, layer=1)
    for r, (k, v) in enumerate(kv):
        check_row(got[r], q[r], k, v, scale, f"row {r}, {lengths[r]} tokens")
    assert ops.device_error() == 0


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("size", [2.0 ** -30, 1e-4, 30.0, 3e4])
def test_attention_of_small_and_large_values(size, dtype):
    """Queries far from one, keys with the inverse size: nothing under- or overflows on the way."""
    g = gen(7)
    lengths = [200, 3]
    c, table, kv = filled(g, lengths, 2, 16, 64, dtype)
    inv = min(1.0 / size, 3e4) if dtype == F16 else 1.0 / size
    for t in (c.k,):
        t *= inv if size > 1 else 1.0
    kv = [((k * inv if size > 1 else k), v) for k, v in kv]
    q = size * normal(g, 2, 8, 64)
    scale = 0.125 if size > 1 else min(0.125 / size, 1e30)
    got = attend(c, table, q, i32(lengths), scale)
    for r, (k, v) in enumerate(kv):
        check_row(got[r], q[r], k, v, scale)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_one_key_far_above_the_others(dtype):
    """Its weight is one to the last bit; the others underflow."""
    g = gen(8)
    c, table, kv = filled(g, [600], 2, 16, 64, dtype)
    q = normal(g, 1, 4, 64)
    scale = 4.0
    for pos in (0, 599, 300):
        k = kv[0][0].clone()
        k[pos] = 5 * torch.stack([q[0, 0], q[0, 2]]).to(dtype)
        for j in range(2):
            c.k[0, table[0, pos // 16].long(), j, pos % 16] = k[pos, j]
        got = attend(c, table, q, i32([600]), scale)
        check_row(got[0], q[0], k, kv[0][1], scale, f"at {pos}")
        for j in range(2):
            assert torch.equal(got[0, 2 * j], kv[0][1][pos, j].float())
        for j in range(2):
            c.k[0, table[0, pos // 16].long(), j, pos % 16] = kv[0][0][pos, j]


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_infinities_and_nan_of_live_tokens(dtype):
    """One in a key or a value reaches its own head's outputs, and no other's."""
    g = gen(9)
    c, table, kv = filled(g, [100, 100, 100, 100], 2, 16, 64, dtype)
    q = normal(g, 4, 4, 64)
    for r, (t, x) in enumerate(((c.k, math.inf), (c.k, math.nan), (c.v, math.nan), (c.v, -math.inf))):
        t[0, table[r, 3].long(), 0, 2, 5] = x
    got = attend(c, table, q, i32([100] * 4), 0.125)
    assert got[1, :2].isnan().all()
    for r in (2, 3):
        assert not torch.isfinite(got[r, :2, 5]).any() and torch.isfinite(got[r, :2, :5]).all()
    for r in range(4):
        check_row(got[r, 2:], q[r, 2:], kv[r][0][:, 1:], kv[r][1][:, 1:], 0.125)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_prompt_rows_share_a_sequence(dtype):
    """Rows of one sequence with lengths 1..m: causal attention; strided q and out; a smaller call in a larger
    workspace; table rows in another order."""
    g = gen(10)
    heads, group, dim, m = 2, 4, 64, 70
    c, table, kv = filled(g, [5, m], heads, 16, dim, dtype)
    wide = normal(g, m, heads * group * dim + 2 * heads * dim)
    q = wide[:, :heads * group * dim].view(m, heads * group, dim)
    out_wide = torch.full_like(wide, math.nan)
    out = out_wide[:, :heads * group * dim].view(m, heads * group, dim)
    ws = ops.paged_attention_workspace(c, 200, heads * group)
    ops.paged_attention(out, q, c, 0, table, i32(list(range(1, m + 1))), 0.125, ws, seq=i32([1] * m))
    assert out_wide[:, heads * group * dim:].isnan().all()
    for r in range(m):
        check_row(out[r], q[r], kv[1][0][:r + 1], kv[1][1][:r + 1], 0.125)
    got = attend(c, table[:, :4], q[:2], i32([5, 64]), 0.125, seq=i32([0, 1]), ws=ws)
    check_row(got[0], q[0], *kv[0], 0.125)
    check_row(got[1], q[1], kv[1][0][:64], kv[1][1][:64], 0.125)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_attention_led_outside_the_cache(dtype):
    """Bad pages, sequences and lengths are skipped and reported, never followed."""
    g = gen(11)
    c, table, kv = filled(g, [100, 100, 100], 2, 16, 64, dtype)
    q = normal(g, 3, 8, 64)
    bad = table.clone()
    bad[0, 2], bad[1, 0], bad[1, 6] = c.pages, -5, 2 ** 31 - 1
    got = attend(c, bad, q, i32([100, 100, 100]), 0.125)
    assert ops.device_error() == 6
    gone = ([t for t in range(100) if t // 16 != 2], list(range(16, 96)), list(range(100)))
    for r in range(3):
        check_row(got[r], q[r], kv[r][0][gone[r]], kv[r][1][gone[r]], 0.125)
    got = attend(c, table[:, :4], q, i32([2 ** 31 - 1, 64, -3]), 0.125)
    assert ops.device_error() == 6
    for r, n in enumerate((64, 64, 0)):
        check_row(got[r], q[r], kv[r][0][:n], kv[r][1][:n], 0.125)
    got = attend(c, table, q, i32([100, 100, 100]), 0.125, seq=i32([-1, 3, 2]))
    assert ops.device_error() == 6
    assert (got[:2] == 0).all()
    check_row(got[2], q[2], *kv[2], 0.125)
    got = attend(c, table, q, i32([0, 0, 100]), 0.125, seq=i32([-1, 3, 2]))  # rows not in use need no sequence
    assert ops.device_error() == 0 and (got[:2] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_offsets_beyond_32_bits(dtype):
    """Two layers of a cache whose pages lie more than 2^31 elements apart."""
    g = gen(12)
    pages, heads, page, dim = 5, 1, 16, 64
    apart = (1 << 29) + 1024
    room = torch.empty(pages * apart + 4096, dtype=dtype, device="cuda")
    shape, strides = (2, pages, heads, page, dim), (2048, apart, page * dim, dim, 1)
    c = ops.KvCache(room.as_strided(shape, strides), room.as_strided(shape, strides, page * dim))
    c.k.fill_(math.nan)
    c.v.fill_(math.nan)
    k, v = normal(g, 70, heads, dim), normal(g, 70, heads, dim)
    table = i32([[4, 2, 3, 1, 0]])
    q = normal(g, 70, 4, dim)
    ops.rope_append(q.clone(), q, k, v, c, 1, torch.arange(70, device="cuda", dtype=torch.int32), table, None,
                    seq=i32([0] * 70))
    k, v = k.to(dtype), v.to(dtype)
    for t in (0, 15, 16, 69):
        p = table[0, t // 16].long()
        assert torch.equal(c.k[1, p, 0, t % 16], k[t, 0]) and torch.equal(c.v[1, p, 0, t % 16], v[t, 0])
    got = attend(c, table, q[:1], i32([70]), 0.125, layer=1)
    check_row(got[0], q[0], k, v, 0.125)
    assert c.k[0].isnan().all() and c.v[0].isnan().all()
    # the fifth page, 2^31 elements from the first, onto a free one and back
    c.k[:, 0], c.v[:, 0] = math.nan, math.nan
    ops.kv_copy_pages(c, i32([4]), i32([0]))
    assert torch.equal(c.k[1, 0], c.k[1, 4]) and torch.equal(c.v[1, 0], c.v[1, 4])
    assert ops.device_error() == 0


# ---- rope_append -------------------------------------------------------------
def rope64(x, pos, turns, interleaved, norm, eps, amplitude):
    """(rotated, |a| + |b| of each value's pair) in 64 bits."""
    x = x.double()
    if norm is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * norm.double()
    size, y = x.abs(), x.clone()
    n = 0 if turns is None else turns.numel()
    if n:
        i = torch.arange(n, device=x.device)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        angle = 2 * math.pi * torch.frac(pos.double()[:, None] * turns)[:, None]
        cos, sin = amplitude * torch.cos(angle), amplitude * torch.sin(angle)
        y[..., a] = x[..., a] * cos - x[..., b] * sin
        y[..., b] = x[..., b] * cos + x[..., a] * sin
        both = abs(amplitude) * (x[..., a].abs() + x[..., b].abs())
        size[..., a], size[..., b] = both, both
    return y, size


def check_rope(got, x, pos, turns, interleaved, norm, eps=1e-5, amplitude=1.0):
    want, size = rope64(x, pos, turns, interleaved, norm, eps, amplitude)
    half_step = 0.0 if got.dtype == F32 else torch.finfo(got.dtype).eps / 2
    least = 0.0 if got.dtype == F32 else torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2
    bound = 32 * U * size
    bound = bound + half_step * (want.abs() + bound) + least
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all() and (err <= bound).all(), (err / bound.clamp_min(1e-300)).max()


# tokens, first position, kv_heads, group, dim, rot, page, interleaved, norm
ROPE = [
    (1, 53, 8, 4, 64, 64, 16, False, False), (5, 0, 2, 3, 128, 128, 16, False, True),
    (64, 2 ** 31 - 4096, 1, 1, 64, 64, 64, False, False), (33, 131000, 8, 3, 128, 64, 16, False, True),
    (40, 17, 5, 7, 80, 36, 24, True, True), (7, 100000, 2, 2, 256, 256, 8, True, False),
    (9, 1, 1, 4, 8, 2, 1, True, False), (12, 3, 3, 1, 96, 70, 7, False, True), (300, 5, 2, 8, 96, 96, 32, True, True),
    (3, 9, 2, 4, 64, 0, 16, False, True), (4, 9, 2, 4, 64, 0, 16, False, False),
    (2000, 5000, 4, 2, 64, 64, 16, False, False),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", range(len(ROPE)))
def test_append(case, dtype):
    m, first, heads, group, dim, rot, page, interleaved, norm = ROPE[case]
    g = gen(200 + case)
    layout, amplitude = ("heads", 1.0) if case % 2 else ("tokens", 1.25)
    hq = heads * group
    # one fused projection's rows
    wide = normal(g, m, (hq + 2 * heads) * dim + 4)
    q = wide[:, :hq * dim].view(m, hq, dim)
    k = wide[:, hq * dim:(hq + heads) * dim].view(m, heads, dim)
    v = wide[:, (hq + heads) * dim:(hq + 2 * heads) * dim].view(m, heads, dim)
    q_norm, k_norm = (1 + 0.1 * normal(g, dim) for _ in range(2)) if norm else (None, None)
    pos = torch.arange(first, first + m, device="cuda", dtype=torch.int32)
    pos[m // 2] = -1 if m > 2 else pos[m // 2]  # a padded token
    pages = -(-m // page) + 2
    c = empty_cache(2, pages, heads, page, dim, dtype, layout)
    # the sequence's table: only the columns of the positions in use are looked at
    cols = (first + m - 1) // page + 1
    table = (torch.arange(cols, device="cuda", dtype=torch.int32) % pages)[None]
    turns = ops.rope_turns(rot, scaling="llama3", factor=32.0) if rot else None
    out, check = guarded(m, hq * dim)
    out = out.view(m, hq, dim)
    before = wide.clone()
    ops.rope_append(out, q, k, v, c, 1, pos, table, turns, seq=i32([0] * m), interleaved=interleaved,
                    amplitude=amplitude, q_norm=q_norm, k_norm=k_norm)
    torch.cuda.synchronize()
    check()
    assert torch.equal(wide, before)
    live = (pos >= 0).nonzero().flatten()
    for t in set(range(m)) - set(live.tolist()):
        assert out[t].isnan().all()  # left as it was
    at = pos[live].long()
    check_rope(out[live], q[live], at, turns, interleaved, q_norm, amplitude=amplitude)
    p, s = table[0].long()[at // page], at % page
    check_rope(c.k[1, p, :, s], k[live], at, turns, interleaved, k_norm, amplitude=amplitude)
    assert torch.equal(c.v[1, p, :, s], v[live].to(dtype))
    # nothing else of the cache is touched
    c.k[1, p, :, s] = math.nan
    c.v[1, p, :, s] = math.nan
    assert c.k.isnan().all() and c.v.isnan().all()
    # in place
    ops.rope_append(q, q, k, v, c, 0, pos, table, turns, seq=i32([0] * m), interleaved=interleaved,
                    amplitude=amplitude, q_norm=q_norm, k_norm=k_norm)
    assert torch.equal(q[live], out[live]) and torch.equal(wide[:, hq * dim:], before[:, hq * dim:])
    assert ops.device_error() == 0


def test_append_led_outside_the_cache():
    g = gen(13)
    m, heads, dim = 7, 2, 64
    q, k, v = normal(g, m, 8, dim), normal(g, m, heads, dim), normal(g, m, heads, dim)
    c = empty_cache(1, 6, heads, 16, dim, BF16)
    table = i32([[0, 1], [2, 6], [-1, 3]])
    pos, seq = i32([5, 16, 20, 3, 40, 2, 17]), i32([0, 0, 1, 2, 0, 3, 2])
    turns = ops.rope_turns(dim)
    out = torch.full_like(q, math.nan)
    ops.rope_append(out, q, k, v, c, 0, pos, table, turns, seq=seq)
    assert ops.device_error() == 6
    check_rope(out, q, pos.long(), turns, False, None)
    written = {0: (0, 5), 1: (1, 0), 6: (3, 1)}
    for t, (p, s) in written.items():
        assert torch.equal(c.v[0, p, :, s], v[t].to(BF16))
        c.k[0, p, :, s] = c.v[0, p, :, s] = math.nan
    assert c.k.isnan().all() and c.v.isnan().all()


def test_norms_of_tiny_and_huge_heads():
    """A head of zeros stays zero; the norm's root is of the mean plus eps."""
    g = gen(14)
    q = normal(g, 3, 2, 64)
    q[0], q[1] = 0.0, q[1] * 1e-3
    q[2] *= 1e6
    k = q[:, :1].clone()
    c = empty_cache(1, 1, 1, 16, 64, F32)
    w = 1 + 0.1 * normal(g, 64)
    out = torch.empty_like(q)
    pos = i32([0, 1, 2])
    ops.rope_append(out, q, k, k, c, 0, pos, i32([[0]]), None, seq=i32([0, 0, 0]), q_norm=w, k_norm=w, eps=1e-6)
    assert (out[0] == 0).all()
    check_rope(out, q, pos.long(), None, False, w, eps=1e-6)
    check_rope(c.k[0, 0, 0, :3][:, None], k, pos.long(), None, False, w, eps=1e-6)


# ---- kv_copy_pages -----------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("layers,pages,heads,page,dim,layout", [
    (1, 2, 1, 1, 8, "heads"), (16, 9, 8, 16, 64, "heads"), (3, 40, 5, 24, 80, "tokens"), (2, 30, 2, 7, 256, "heads"),
    (28, 300, 8, 16, 128, "heads"), (1, 5, 1, 128, 96, "side")])
def test_copy_pages(layers, pages, heads, page, dim, layout, dtype):
    g = gen(300 + pages)
    if layout == "side":  # keys and values of a slot side by side
        t = normal(g, layers, pages, heads, page, 2, dim).to(dtype)
        c = ops.KvCache(t[..., 0, :], t[..., 1, :])
    else:
        c = empty_cache(layers, pages, heads, page, dim, dtype, layout)
        for x in (c.k, c.v):
            x.copy_(normal(g, *x.shape))
    k, v = c.k.clone(), c.v.clone()
    mixed = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    n = pages // 2
    src, dst = mixed[:n].clone(), mixed[n:2 * n].clone()
    src[n // 2] = src[0]  # one page to two places
    k[:, dst.long()], v[:, dst.long()] = k[:, src.long()], v[:, src.long()]
    ops.kv_copy_pages(c, src, dst)
    assert torch.equal(c.k, k) and torch.equal(c.v, v)
    # padding is skipped without a word; pages outside are skipped and reported
    ops.kv_copy_pages(c, i32([-1, 0, -1]), i32([0, -1, -1]))
    assert ops.device_error() == 0
    ops.kv_copy_pages(c, i32([pages, 0]), i32([0, 2 ** 31 - 1]))
    assert ops.device_error() == 6
    assert torch.equal(c.k, k) and torch.equal(c.v, v)


# ---- together ----------------------------------------------------------------
class Decoder:
    """One attention block's int8 projections beside a paged cache, and the same in 64 bits."""

    def __init__(self, g, dim_model=512, heads=8, kv_heads=2, dim=64, dtype=BF16, layout="heads"):
        self.heads, self.kv_heads, self.dim, self.model = heads, kv_heads, dim, dim_model
        self.rows = (heads + 2 * kv_heads) * dim
        self.w = [self.quantised(g, self.rows, dim_model), self.quantised(g, dim_model, heads * dim)]
        self.turns = ops.rope_turns(dim, scaling="llama3", factor=32.0)
        self.norms = [1 + 0.1 * normal(g, dim) for _ in range(2)]
        self.kv = PagedKvCache(layers=1, pages=64, kv_heads=kv_heads, head_dim=dim, max_seqs=16, dtype=dtype,
                               layout=layout)
        self.ws = ops.paged_attention_workspace(self.kv.cache, 64, heads)

    @staticmethod
    def quantised(g, rows, cols):
        w = 0.05 * normal(g, rows, cols)
        q, s = torch.empty(rows, cols, dtype=torch.int8, device="cuda"), torch.empty(rows, cols // 64, device="cuda")
        ops.quantize_weights(q, s, w, rows, cols)
        return q, s

    def project(self, x, which):
        q, s = self.w[which]
        m, (rows, cols) = x.shape[0], q.shape
        y = torch.empty(m, rows, device="cuda")
        if m == 1:
            ops.matmul_int8(y, x, q, s, cols, rows)
        else:
            xq, xs = torch.empty(m, cols, dtype=torch.int8, device="cuda"), torch.empty(m, device="cuda")
            ops.quantize_activation_rows(xq, xs, x, m, cols)
            ops.gemm_w8a8(y, xq, xs, q, s, m, cols, rows)
        return y

    def split(self, y):
        a, b = self.heads * self.dim, (self.heads + self.kv_heads) * self.dim
        return (y[:, :a].view(-1, self.heads, self.dim), y[:, a:b].view(-1, self.kv_heads, self.dim),
                y[:, b:].view(-1, self.kv_heads, self.dim))

    def attend(self, y, seq, pos, lengths):
        """From the q/k/v projection's rows to attention's output."""
        q, k, v = self.split(y)
        out = torch.empty(y.shape[0], self.heads * self.dim, device="cuda")
        ops.rope_append(q, q, k, v, self.kv.cache, 0, pos, self.kv.page_table, self.turns, seq=seq,
                        q_norm=self.norms[0], k_norm=self.norms[1])
        ops.paged_attention(out.view(-1, self.heads, self.dim), q, self.kv.cache, 0, self.kv.page_table, lengths,
                            self.dim ** -0.5, self.ws, seq=seq)
        return out

    def step(self, x, seqs):
        """One token of every sequence: the block's output, what it computed, and where the tokens went."""
        pos = [self.kv.length(s) for s in seqs]
        self.kv.extend(seqs)
        y = self.project(x, 0)
        raw = y.clone()
        out = self.attend(y, i32(seqs), i32(pos), i32([p + 1 for p in pos]))
        return self.project(out, 1), raw, out


@pytest.mark.parametrize("dtype,layout", [(F32, "heads"), (BF16, "heads"), (F16, "tokens")])
def test_decode_with_forks_and_compaction(dtype, layout):
    """A prompt of 37 tokens as rows of one call, then decode steps of a growing set of forks, pages freed and
    compacted on the way: every output is the formula's over the sequence's own keys and values."""
    g = gen(15)
    d = Decoder(g, dtype=dtype, layout=layout)
    first = d.kv.new()
    m = 37
    d.kv.extend([first], [m])
    x = normal(g, m, d.model)
    y = d.project(x, 0)
    raw = y.clone()
    at = torch.arange(m, device="cuda", dtype=torch.int32)
    out = d.attend(y, i32([first] * m), at, at + 1)
    scale = d.dim ** -0.5

    def rotated(raw, pos):
        q, k, v = d.split(raw)
        q, _ = rope64(q, pos, d.turns, False, d.norms[0], 1e-5, 1.0)
        k, _ = rope64(k, pos, d.turns, False, d.norms[1], 1e-5, 1.0)
        return q.float(), k, v

    def check(out, q, keys, values):
        # q and k differ from the kernel's by roundings; k by up to one step of the cache's type where a border is near
        want, a, size = attention64(q, keys.to(dtype), values.to(dtype), scale)
        half = torch.finfo(dtype).eps / 2
        n = keys.shape[0]
        slack = (4 * (64 * U + (half if dtype != F32 else 0)) * size[:, None] + (100 + 8 * math.sqrt(n)) * U) * a
        assert ((out.double().view_as(want) - want).abs() <= slack + 1e-30).all()

    q, k, v = rotated(raw, at.long())
    for t in (0, 15, 16, 36):
        check(out[t], q[t], k[:t + 1], v[:t + 1])
    history = {first: (k, v)}
    for step in range(20):
        if step in (1, 4, 5):
            s = list(history)[0]
            new = d.kv.fork(s)
            history[new] = history[s]
        if step == 9:
            gone = list(history)[1]
            d.kv.free(gone)
            del history[gone]
            assert d.kv.compact() > 0
        seqs = list(history)
        x = normal(g, len(seqs), d.model)
        pos = torch.tensor([d.kv.length(s) for s in seqs], device="cuda")
        result, raw, out = d.step(x, seqs)
        q, k, v = rotated(raw, pos)
        for i, s in enumerate(seqs):
            history[s] = tuple(torch.cat((old, new[i:i + 1])) for old, new in zip(history[s], (k, v)))
            check(out[i], q[i], *history[s])
        assert torch.isfinite(result).all()
    assert ops.device_error() == 0


def test_captured_steps_and_other_streams():
    """A step captured once and replayed with other positions, lengths and inputs in the same tensors, on a stream of
    its own, gives an eager step's bits; two captured steps share the workspace."""
    g = gen(16)
    d = Decoder(g)
    seqs = [d.kv.new() for _ in range(4)]
    d.kv.extend(seqs, [40, 3, 64, 17])
    for x in (d.kv.cache.k, d.kv.cache.v):
        x.copy_(normal(g, *x.shape))
    seq, pos, lengths = i32(seqs), i32([0] * 4), i32([1] * 4)
    y, out = torch.zeros(4, d.rows, device="cuda"), torch.empty(4, d.heads * d.dim, device="cuda")
    start = torch.zeros_like(y)

    def step():
        y.copy_(start)
        out.copy_(d.attend(y, seq, pos, lengths))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        graphs.append(graph)
    for k, at in enumerate(([39, 2, 63, 16], [0, 0, 0, 0], [20, 1, 30, 5])):
        start.copy_(normal(g, 4, d.rows))
        pos.copy_(i32(at))
        lengths.copy_(i32([a + 1 for a in at]))
        before = d.kv.cache.k.clone(), d.kv.cache.v.clone()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            graphs[k % 2].replay()
        torch.cuda.current_stream().wait_stream(stream)
        got = out.clone()
        after = d.kv.cache.k.clone(), d.kv.cache.v.clone()
        d.kv.cache.k.copy_(before[0])
        d.kv.cache.v.copy_(before[1])
        step()
        assert torch.equal(got, out) and torch.equal(after[0], d.kv.cache.k) and torch.equal(after[1], d.kv.cache.v)
    assert ops.device_error() == 0


def test_back_to_back_calls_see_each_other():
    """Appends and attentions queued without a wait between them, layer after layer."""
    g = gen(17)
    layers, heads, group, dim, m = 6, 2, 4, 64, 3
    c = empty_cache(layers, 8, heads, 16, dim, BF16, fill=0.0)
    for x in (c.k, c.v):
        x.copy_(normal(g, *x.shape))
    table, lengths = i32([[0, 1], [2, 3], [4, 5]]), i32([20, 32, 1])
    ws = ops.paged_attention_workspace(c, m, heads * group)
    qs = [normal(g, m, heads * group, dim) for _ in range(layers)]
    ks = [normal(g, m, heads, dim) for _ in range(layers)]
    outs = [torch.empty_like(q) for q in qs]
    torch.cuda.synchronize()
    for i in range(layers):
        q = qs[i].clone()
        ops.rope_append(q, q, ks[i], ks[i], c, i, lengths - 1, table, None)
        ops.paged_attention(outs[i], q, c, i, table, lengths, 0.125, ws)
    torch.cuda.synchronize()
    for i in range(layers):
        for r, n in enumerate(lengths.tolist()):
            p = table[r].long()
            k, v = (x[i, p].transpose(1, 2).reshape(-1, heads, dim)[:n] for x in (c.k, c.v))
            assert torch.equal(k[-1], ks[i][r].to(BF16))
            check_row(outs[i][r], qs[i][r], k, v, 0.125)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_attention_in_place(dtype):
    """out is q, over rows that one CTA, several, and none work on."""
    g = gen(19)
    lengths = [9000, 1, 0, 40, 2000]
    c, table, kv = filled(g, lengths, 2, 16, 64, dtype)
    q = normal(g, 5, 8, 64)
    want = attend(c, table, q, i32(lengths), 0.125)
    ws = ops.paged_attention_workspace(c, 5, 8)
    ops.paged_attention(q, q, c, 0, table, i32(lengths), 0.125, ws)
    assert torch.equal(q.view(torch.int32), want.view(torch.int32))


def test_one_workspace_for_calls_of_all_sizes():
    """Calls of other head sizes, row counts and types between two of the same: the same bits."""
    g = gen(20)
    cases = []
    for lengths, heads, group, dim, dtype in (([5000], 8, 8, 256, F32), ([3] * 700, 2, 4, 64, BF16),
                                              ([4000, 17], 4, 5, 128, F16), ([20000], 1, 16, 64, BF16)):
        c, table, kv = filled(g, lengths, heads, 16, dim, dtype)
        cases.append((c, table, kv, normal(g, len(lengths), heads * group, dim), i32(lengths), lengths))
    ws = max((ops.paged_attention_workspace(c, q.shape[0], q.shape[1]) for c, _, _, q, _, _ in cases), key=len)
    seen = {}
    for turn in (0, 1, 2, 3, 1, 0, 3, 2):
        c, table, kv, q, lengths, plain = cases[turn]
        got = attend(c, table, q, lengths, q.shape[2] ** -0.5, ws=ws)
        if turn in seen:
            assert torch.equal(got.view(torch.int32), seen[turn].view(torch.int32))
        else:
            seen[turn] = got
            for r in (0, len(plain) - 1):
                check_row(got[r], q[r], *kv[r], q.shape[2] ** -0.5)


def test_many_short_rows():
    """More rows than threads, some without tokens, all of one sequence."""
    g = gen(21)
    c, table, kv = filled(g, [70], 2, 16, 64, BF16)
    rows = 3001
    lengths = [(7 * r) % 71 for r in range(rows)]
    q = normal(g, rows, 4, 64)
    got = attend(c, table, q, i32(lengths), 0.125, seq=torch.zeros(rows, dtype=torch.int32, device="cuda"))
    for r in list(range(0, rows, 97)) + [rows - 1]:
        check_row(got[r], q[r], kv[0][0][:lengths[r]], kv[0][1][:lengths[r]], 0.125, f"row {r}")
    empty = torch.tensor([n == 0 for n in lengths], device="cuda")
    assert (got[empty] == 0).all() and ops.device_error() == 0


def test_two_streams_at_once():
    """Two calls under way at once, each with its own workspace, on streams that are not the current one."""
    g = gen(22)
    c, table, kv = filled(g, [3000, 2500, 100], 2, 16, 64, BF16)
    qs = [normal(g, 3, 8, 64) for _ in range(2)]
    lengths = i32([3000, 2500, 100])
    want = [attend(c, table, q, lengths, 0.125) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    ws = [ops.paged_attention_workspace(c, 3, 8) for _ in range(2)]
    outs = [torch.empty_like(q) for q in qs]
    torch.cuda.synchronize()
    for _ in range(10):
        for i in range(2):
            ops.paged_attention(outs[i], qs[i], c, 0, table, lengths, 0.125, ws[i], stream=streams[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(outs[i].view(torch.int32), want[i].view(torch.int32))


def test_refusals_name_the_call():
    g = gen(18)
    c, table, _ = filled(g, [20], 2, 16, 64, BF16)
    q = normal(g, 1, 8, 64)
    ws = ops.paged_attention_workspace(c, 1, 8)
    with pytest.raises(MliError, match="paged_attention: invalid argument"):
        ops.paged_attention(q, q, c, 1, table, i32([20]), 0.125, ws)
    with pytest.raises(MliError, match="paged_attention: invalid argument"):
        ops.paged_attention(q, q, c, 0, table, i32([20]), 0.125, ws[:8])
    with pytest.raises(MliError, match="paged_attention: invalid argument"):
        ops.paged_attention(q[:, :7], q[:, :7], c, 0, table, i32([20]), 0.125, ws)
    with pytest.raises(MliError, match="rope_append: invalid argument"):
        ops.rope_append(q, q, q[:, :2], q[:, :2], c, 0, i32([3]), table, ops.rope_turns(66))
    with pytest.raises(MliError, match="kv_copy_pages: invalid argument"):
        ops.kv_copy_pages(c, i32([]), i32([]))
    with pytest.raises(ValueError):
        ops.paged_attention_workspace(c, 1, 7)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("power", [-118, -86, -75, -62, 100, 126])
@pytest.mark.parametrize("group,dim", [(4, 64), (8, 128), (2, 256)])
def test_attention_of_queries_of_every_size(group, dim, power, dtype):
    """Queries from near the least normal number to the largest one, with the scale that makes ordinary scores of them:
    as exact as any others."""
    g = gen(30)
    lengths = [150, 3]
    c, table, kv = filled(g, lengths, 2, 16, dim, dtype)
    small = 2.0 ** -10 if power > 0 else 1.0  # keys, so that no score overflows
    c.k.mul_(small)
    kv = [(k * small, v) for k, v in kv]
    q = normal(g, 2, 2 * group, dim).clamp(-3.9, 3.9) * 2.0 ** power
    if power == 126:
        q[0, 0, 0] = torch.finfo(F32).max
    scale = dim ** -0.5 / (2.0 ** power * small)
    got = attend(c, table, q, i32(lengths), scale)
    for r, (k, v) in enumerate(kv):
        check_row(got[r], q[r], k, v, scale, f"row {r}")


@pytest.mark.parametrize("dtype,dim", [(F16, 8), (F32, 4)])
def test_a_page_table_that_names_2_to_the_31_tokens(dtype, dim):
    """Two rows of a table of 2049 columns, all the same page of 2^20 slots.  A length above 2^31 - 64 is cut to that and
    reported; the row beside it is as ever.  Equal weights, and values of one in the first half of the page, of zero in
    the second: sums of whole numbers, below 2^24 units in a CTA and so exact; the joins of all CTAs round output and
    sum once each, so a half comes out to 2 sm_count u and a few for the quotient."""
    size, sms = 1 << 20, torch.cuda.get_device_properties(0).multi_processor_count
    c = empty_cache(1, 1, 1, size, dim, dtype, fill=0.0)
    c.v[0, 0, 0, :size // 2] = 1.0
    table = torch.zeros(2, 2049, dtype=torch.int32, device="cuda")
    q = torch.zeros(2, 1, dim, device="cuda")
    q[1] = 1.0
    for length, error in ((2 ** 31 - 64, 0), (2 ** 31 - 63, 6), (2 ** 31 - 1, 6)):
        got = attend(c, table, q, i32([length, 5]), 0.5)
        assert ops.device_error() == error
        assert (got[0] - 0.5).abs().max() <= (2 * sms + 8) * U and (got[1] == 1.0).all()


@pytest.mark.parametrize("first", [0, 131072 - 2000, 2 ** 31 - 2000])
@pytest.mark.parametrize("amplitude", [1.0, 1.25])
def test_cosines_and_sines_are_exact_to_their_last_bits(first, amplitude):
    """Pairs (1, 0) become (cos, sin) of the angle, held against the angle taken from pos * turns in whole numbers.
    sincospi is off by a unit in the last place (2 u), twice over where the angle's rest that fp32 does not hold cancels
    half of it; that rest's own roundings (3 u) and the sum's (u) follow, and the amplitude's (u): below 12 u of the value
    itself, however near a quarter turn the angle is, and the angle itself is held to 2^-53 of a half turn."""
    g = gen(32)
    m, dim = 1999, 64
    pos = torch.arange(first, first + m, device="cuda", dtype=torch.int32)
    turns = ops.rope_turns(dim)
    turns[0], turns[1] = 0.25, 0.25 + 2.0 ** -40  # exact quarters, and next to them
    q = torch.zeros(m, 1, dim, device="cuda")
    q[..., 0::2] = 1.0
    c = empty_cache(1, 1, 1, 1, dim, F32)
    out, kv = torch.empty_like(q), normal(g, m, 1, dim)
    table = torch.full((1, 1), -1, dtype=torch.int32, device="cuda")  # only the queries are looked at
    ops.rope_append(out, q, kv, kv, c, 0, pos, table, turns, seq=i32([0] * m), interleaved=True, amplitude=amplitude)
    assert ops.device_error() == 6
    got = out[:, 0].double().cpu().numpy().reshape(m, dim // 2, 2)
    want = np.empty_like(got)
    for i, t in enumerate(turns.tolist()):
        num, den = t.as_integer_ratio()
        for j in range(m):
            # the angle less its nearest quarter turn, in whole numbers: num / (4 den) turns
            part = 4 * (first + j) * num
            quarter = (2 * part + den) // (2 * den)
            x = 2 * math.pi * ((part - quarter * den) / den) / 4
            co, si = math.cos(x), math.sin(x)
            want[j, i] = ((co, si), (-si, co), (-co, -si), (si, -co))[quarter % 4]
    want *= amplitude
    err = np.abs(got - want)
    assert (err <= 12 * U * np.abs(want) + 2.0 ** -50).all(), (err / (12 * U * np.abs(want) + 2.0 ** -50)).max()


@pytest.mark.parametrize("dim,tokens,tile,side", [(64, 8192, 32, 2), (128, 4096, 16, 1), (256, 4096, 8, 1)])
@pytest.mark.parametrize("group", [1, 5])
def test_fp32_outputs_are_summed_tile_by_tile(dim, tokens, tile, side, group):
    """Equal weights and equal values, whose running fp32 sum would lose the same half step with every token from 2048
    on: as many rows as there are warps, so that each sums a row alone.  A tile's sum takes tile / side roundings, the
    sum of the tiles one each, lanes, quotient and product four: each at most u of a sum of positive numbers."""
    rows = 8 * torch.cuda.get_device_properties(0).multi_processor_count
    value = 1 + 2.0 ** -13 - 2.0 ** -20
    c = empty_cache(1, tokens // 64, 1, 64, dim, F32, fill=value)
    table = torch.arange(tokens // 64, device="cuda", dtype=torch.int32)[None]
    q = torch.zeros(rows, group, dim, device="cuda")
    got = attend(c, table, q, i32([tokens] * rows), 0.125, seq=i32([0] * rows))
    value = float(c.v[0, 0, 0, 0, 0])
    err = (got.double() - value).abs().max().item()
    assert err <= (tile / side + tokens / tile + 4) * U * value, err / (U * value)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_an_infinite_key_makes_a_head_not_finite_or_leaves_its_token_out(dtype):
    """A score of -inf weighs nothing, one of inf or NaN reaches every output of its head: with an fp32 cache by the
    query's sign, with the others by what the parts of the query multiply it to."""
    g = gen(31)
    lengths = [100] * 4
    c, table, kv = filled(g, lengths, 2, 16, 64, dtype)
    q = normal(g, 4, 4, 64)
    for r, x in enumerate((math.inf, math.inf, -math.inf, -math.inf)):
        c.k[0, table[r, 3].long(), 0, 2, 5] = x  # token 50
        q[r, :2, 5] = q[r, :2, 5].abs() * (1 if r % 2 else -1)
    got = attend(c, table, q, i32(lengths), 0.125)
    rest = [t for t in range(100) if t != 50]
    for r in range(4):
        below = (r % 2 == 0) == (r < 2)  # the scores are -inf
        for h in range(2):
            if dtype == F32 or not got[r, h].isfinite().any():
                assert got[r, h].isfinite().all() if dtype == F32 and below else got[r, h].isnan().all()
            if got[r, h].isfinite().any():
                assert below
                check_row(got[r, h:h + 1], q[r, h:h + 1], kv[r][0][rest, :1], kv[r][1][rest, :1], 0.125)
        check_row(got[r, 2:], q[r, 2:], kv[r][0][:, 1:], kv[r][1][:, 1:], 0.125)


def test_pages_do_not_change_within_a_capture():
    """Each of PagedKvCache's changes is refused while the current stream captures, and leaves no trace."""
    kv = PagedKvCache(layers=1, pages=8, kv_heads=2, head_dim=64, page_size=4, max_seqs=3)
    a, b = kv.new(), kv.new()
    kv.extend([a, b], [4, 5])
    kv.free(a)
    a = kv.new()
    x = torch.zeros(4, device="cuda")
    table = kv.page_table.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: kv.extend([b], [4]), lambda: kv.fork(b), lambda: kv.free(b), kv.compact):
            with pytest.raises(RuntimeError, match="capturing"):
                call()
        kv.extend([b], [3])  # no new page
        x.add_(1.0)
    graph.replay()
    assert (x == 1).all() and torch.equal(kv.page_table, table)
    assert kv.length(b) == 8 and len(kv.pages(b)) == 2 and kv.free_pages == 6
    kv.extend([b], [1])
    c = kv.fork(b)
    kv.extend([c])  # pages 1, 2 and 3; page 0 is b's third
    kv.free(b)
    assert kv.compact() == 1 and sorted(kv.pages(c)) == [0, 1, 2]
    assert kv.page_table[c, :3].tolist() == kv.pages(c) and (kv.page_table[c, 3:] == -1).all()
    assert (kv.page_table[[a, b]] == -1).all()
