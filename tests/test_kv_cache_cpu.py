"""The paged key-value cache on the CPU: refusals of the C ABI and of the Python
wrappers (decided before any CUDA call), the rotary frequencies, and the page
bookkeeping of PagedKvCache with the page copy replaced by indexing."""
import ctypes
import math

import numpy as np
import pytest

from minillama_infra_b200 import _lib, ops
from minillama_infra_b200.kv_cache import PagedKvCache

torch = pytest.importorskip("torch")
OK, INVALID, UNSUPPORTED = _lib.MLI_OK, _lib.MLI_ERR_INVALID_ARG, _lib.MLI_ERR_UNSUPPORTED
A = 4096  # stands for an aligned device address; no call here reaches the GPU


def cache(**kw):
    d = dict(k=A, v=A, dtype=2, layers=2, pages=8, page_size=16, kv_heads=4, head_dim=64, layer_stride=8 * 4 * 16 * 64,
             page_stride=4 * 16 * 64, head_stride=16 * 64, slot_stride=64)
    return _lib.KvCacheDesc(**{**d, **kw})


def rope(**kw):
    d = dict(m=3, heads=8, rot_dim=64, interleaved=0, amplitude=1.0, eps=1e-5, turns=A, q_out=A, q=2 * A, k=A, v=A,
             q_out_stride=512, q_stride=512, k_stride=256, v_stride=256, q_norm=None, k_norm=None, pos=A, seq=A,
             page_table=A, table_rows=2, table_cols=4, table_stride=4)
    return _lib.RopeOp(**{**d, **kw})


def attention(**kw):
    d = dict(rows=3, heads=8, scale=0.125, out=A, q=A, out_stride=512, q_stride=512, lengths=A, seq=A, page_table=A,
             table_rows=2, table_cols=4, table_stride=4, workspace=A, workspace_bytes=1 << 30)
    return _lib.AttentionOp(**{**d, **kw})


BAD_CACHES = [(dict(k=None), INVALID), (dict(v=None), INVALID), (dict(dtype=3), INVALID), (dict(dtype=-1), INVALID),
              (dict(layers=0), INVALID), (dict(pages=0), INVALID), (dict(page_size=0), INVALID),
              (dict(kv_heads=0), INVALID), (dict(head_dim=0), INVALID), (dict(page_stride=-64), INVALID),
              (dict(head_dim=60), UNSUPPORTED), (dict(head_dim=264), UNSUPPORTED), (dict(k=A + 8), UNSUPPORTED),
              (dict(v=A + 2), UNSUPPORTED), (dict(slot_stride=68), UNSUPPORTED), (dict(head_stride=1028), UNSUPPORTED),
              (dict(page_stride=4100), UNSUPPORTED), (dict(layer_stride=4), UNSUPPORTED)]


@pytest.mark.parametrize("change,status", BAD_CACHES)
def test_bad_caches_are_refused(change, status):
    l, c = _lib.lib(), cache(**change)
    wide = dict(q_stride=4096, q_out_stride=4096, k_stride=4096, v_stride=4096)
    assert l.mli_rope_append(rope(rot_dim=32, **wide), c, 0, None) == status
    assert l.mli_paged_attention(attention(q_stride=4096, out_stride=4096), c, 0, None) == status
    assert l.mli_kv_copy_pages(c, A, A, 1, None) == status
    assert l.mli_last_status() == status


@pytest.mark.parametrize("change,status", [
    (dict(m=0), INVALID), (dict(heads=6), INVALID), (dict(heads=0), INVALID), (dict(rot_dim=63), INVALID),
    (dict(rot_dim=66), INVALID), (dict(rot_dim=-2), INVALID), (dict(turns=None), INVALID), (dict(q=None), INVALID),
    (dict(q_out=None), INVALID), (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(pos=None), INVALID),
    (dict(page_table=None), INVALID), (dict(seq=None), INVALID), (dict(table_rows=0), INVALID),
    (dict(table_cols=0), INVALID), (dict(table_stride=3), INVALID), (dict(q_stride=508), INVALID),
    (dict(q_out_stride=508), INVALID), (dict(k_stride=252), INVALID), (dict(v_stride=252), INVALID),
    (dict(q_out=2 * A, q_out_stride=516), INVALID), (dict(amplitude=math.inf), INVALID),
    (dict(q_norm=A, eps=math.nan), INVALID), (dict(k_norm=A, eps=-1.0), INVALID),
    (dict(q=2 * A + 4), UNSUPPORTED), (dict(q_out=A + 8), UNSUPPORTED), (dict(k=A + 4), UNSUPPORTED),
    (dict(v=A + 4), UNSUPPORTED), (dict(q_stride=514), UNSUPPORTED), (dict(k_norm=A + 4), UNSUPPORTED)])
def test_bad_appends_are_refused(change, status):
    assert _lib.lib().mli_rope_append(rope(**change), cache(), 0, None) == status


@pytest.mark.parametrize("change,status", [
    (dict(rows=0), INVALID), (dict(rows=-1), INVALID), (dict(heads=6), INVALID), (dict(scale=0.0), INVALID),
    (dict(scale=-1.0), INVALID), (dict(scale=math.nan), INVALID), (dict(scale=math.inf), INVALID),
    (dict(out=None), INVALID), (dict(q=None), INVALID), (dict(lengths=None), INVALID),
    (dict(page_table=None), INVALID), (dict(seq=None), INVALID), (dict(table_stride=3), INVALID),
    (dict(table_cols=0), INVALID), (dict(workspace=None), INVALID), (dict(workspace_bytes=15), INVALID),
    (dict(q_stride=508), INVALID), (dict(out_stride=508), INVALID), (dict(q=A + 4), UNSUPPORTED),
    (dict(out=A + 4), UNSUPPORTED), (dict(out_stride=514), UNSUPPORTED), (dict(workspace=A + 8), UNSUPPORTED)])
def test_bad_attentions_are_refused(change, status):
    assert _lib.lib().mli_paged_attention(attention(**change), cache(), 0, None) == status


def test_layers_null_structs_and_counts_are_refused():
    l, c = _lib.lib(), cache()
    for layer in (-1, 2):
        assert l.mli_rope_append(rope(), c, layer, None) == INVALID
        assert l.mli_paged_attention(attention(), c, layer, None) == INVALID
    assert l.mli_rope_append(None, c, 0, None) == INVALID
    assert l.mli_rope_append(rope(), None, 0, None) == INVALID
    assert l.mli_paged_attention(None, c, 0, None) == INVALID
    assert l.mli_paged_attention(attention(), None, 0, None) == INVALID
    assert l.mli_kv_copy_pages(None, A, A, 1, None) == INVALID
    assert l.mli_kv_copy_pages(c, None, A, 1, None) == INVALID
    assert l.mli_kv_copy_pages(c, A, None, 1, None) == INVALID
    assert l.mli_kv_copy_pages(c, A, A, 0, None) == INVALID


def test_sizes_beyond_the_kernels_counters_are_refused():
    """More tiles than an int counts; pages of more 16-byte pieces than one does; more layers than a grid has."""
    l, c = _lib.lib(), cache()
    wide = dict(table_cols=1 << 27, table_stride=1 << 27)  # of 64 tokens a tile: 2^25 tiles a row and head
    assert l.mli_paged_attention(attention(rows=1 << 10, **wide), c, 0, None) == UNSUPPORTED
    assert l.mli_paged_attention(attention(rows=1 << 20, table_cols=1 << 13, table_stride=1 << 13), c, 0, None) == UNSUPPORTED
    assert l.mli_kv_copy_pages(cache(page_size=1 << 23), A, A, 1, None) == UNSUPPORTED
    assert l.mli_kv_copy_pages(cache(layers=65536), A, A, 1, None) == UNSUPPORTED


def test_workspace_bytes():
    size = _lib.lib().mli_paged_attention_workspace_bytes
    assert size(1, 8, 8, 64) > 0
    assert size(64, 32, 8, 128) >= size(1, 32, 8, 128)
    for args in ((0, 8, 8, 64), (1, 0, 8, 64), (1, 8, 0, 64), (1, 9, 8, 64), (1, 8, 8, 0), (1, 8, 8, 257)):
        assert size(*args) == 0


# ---- rotary frequencies ------------------------------------------------------
def frequency(i, rot, theta, scaling, factor, low, high, length):
    f = theta ** (-2 * i / rot)
    if scaling == "linear":
        return f / factor
    if scaling == "llama3":  # src/model_cuda_v2_shared.cu:233-250
        wave = 2 * math.pi / f
        if wave > length / low:
            return f / factor
        if wave < length / high:
            return f
        mix = (length / wave - low) / (high - low)
        return (1 - mix) * f / factor + mix * f
    if scaling == "yarn":
        at = [rot * math.log(length / (r * 2 * math.pi)) / (2 * math.log(theta)) for r in (high, low)]
        a, b = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
        ramp = min(1.0, max(0.0, (i - a) / max(b - a, 1e-3)))
        return f / factor * ramp + f * (1 - ramp)
    return f


@pytest.mark.parametrize("rot,theta,scaling,factor,low,high,length", [
    (64, 500000.0, "none", 1.0, 1.0, 4.0, 8192), (2, 10000.0, "none", 1.0, 1.0, 4.0, 8192),
    (128, 500000.0, "llama3", 32.0, 1.0, 4.0, 8192), (64, 500000.0, "llama3", 32.0, 1.0, 4.0, 8192),
    (36, 10000.0, "linear", 4.0, 1.0, 4.0, 4096), (128, 10000.0, "yarn", 16.0, 1.0, 32.0, 4096),
    (256, 1000000.0, "yarn", 4.0, 1.0, 32.0, 32768)])
def test_rope_turns(rot, theta, scaling, factor, low, high, length):
    got = ops.rope_turns(rot, theta, scaling, factor, low, high, length, device="cpu")
    want = [frequency(i, rot, theta, scaling, factor, low, high, length) / (2 * math.pi) for i in range(rot // 2)]
    # pow, a few products and a quotient in 64 bits: each within a few units of 2^-53
    assert got.dtype == torch.float64 and np.allclose(got.numpy(), want, rtol=2.0 ** -46, atol=0)


@pytest.mark.parametrize("args", [
    (0, 1e4, 0, 1.0, 1.0, 4.0, 8192), (63, 1e4, 0, 1.0, 1.0, 4.0, 8192), (64, 0.0, 0, 1.0, 1.0, 4.0, 8192),
    (64, math.nan, 0, 1.0, 1.0, 4.0, 8192), (64, 1e4, 4, 1.0, 1.0, 4.0, 8192), (64, 1e4, -1, 1.0, 1.0, 4.0, 8192),
    (64, 1e4, 1, 0.0, 1.0, 4.0, 8192), (64, 1e4, 2, 8.0, 4.0, 4.0, 8192), (64, 1e4, 2, 8.0, 1.0, 4.0, 0),
    (64, 1e4, 3, 8.0, 0.0, 4.0, 8192), (64, 1.0, 3, 8.0, 1.0, 32.0, 8192)])
def test_bad_rope_turns_are_refused(args):
    out = (ctypes.c_double * 64)()
    assert _lib.lib().mli_rope_turns(out, *args) == INVALID
    assert _lib.lib().mli_rope_turns(None, 64, 1e4, 0, 1.0, 1.0, 4.0, 8192) == INVALID


def test_rope_turns_names():
    with pytest.raises(ValueError):
        ops.rope_turns(64, scaling="ntk", device="cpu")


# ---- wrappers ------------------------------------------------------------------
def test_cache_handle():
    t = torch.zeros(2, 5, 16, 4, 2, 64, dtype=torch.float16)  # keys and values of a page side by side, token-major
    c = ops.KvCache(t[..., 0, :].transpose(2, 3), t[..., 1, :].transpose(2, 3))
    d = c.desc
    assert (d.layers, d.pages, d.kv_heads, d.page_size, d.head_dim, d.dtype) == (2, 5, 4, 16, 64, 1)
    assert (d.layer_stride, d.page_stride, d.head_stride, d.slot_stride) == (5 * 8192, 8192, 128, 512)
    assert d.v - d.k == 128
    one = ops.KvCache(torch.zeros(1, 1, 1, 3, 64), torch.zeros(1, 1, 1, 3, 64)).desc
    assert (one.layer_stride, one.page_stride, one.head_stride, one.slot_stride) == (0, 0, 0, 64)
    k = torch.zeros(1, 2, 4, 16, 64)
    for bad in (k[0], k[..., :32], k.half(), k.transpose(2, 3).contiguous().transpose(2, 3)):
        with pytest.raises(ValueError):
            ops.KvCache(k, bad)
    for bad in (k.double(), k.transpose(3, 4)):
        with pytest.raises(ValueError):
            ops.KvCache(bad, bad.clone(memory_format=torch.preserve_format))


def test_wrappers_refuse_host_tensors_and_wrong_shapes():
    k = torch.zeros(1, 2, 4, 16, 64)
    c = ops.KvCache(k, k.clone())
    q, kv = torch.zeros(3, 8, 64), torch.zeros(3, 4, 64)
    ints, table = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32)
    turns, ws = ops.rope_turns(64, device="cpu"), torch.zeros(64, dtype=torch.uint8)

    def append(**kw):
        a = dict(q_out=q.clone(), q=q, k=kv, v=kv, cache=c, layer=0, pos=ints, page_table=table, turns=turns)
        ops.rope_append(**{**a, **kw})

    def attend(**kw):
        a = dict(out=q.clone(), q=q, cache=c, layer=0, page_table=table, lengths=ints, scale=0.125, workspace=ws)
        ops.paged_attention(**{**a, **kw})

    for kw in (dict(), dict(q=q.half()), dict(k=kv[:2]), dict(v=q), dict(pos=ints.long()), dict(turns=turns.float()),
               dict(page_table=table.long()), dict(page_table=table[0]), dict(seq=ints[:2]), dict(q_norm=q[0, 0, :32]),
               dict(q=q.transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(ValueError):
            append(**kw)
    for kw in (dict(), dict(out=q.half()), dict(lengths=ints[:2]), dict(workspace=q), dict(q=q[:, :, :32]),
               dict(page_table=table.T)):
        with pytest.raises(ValueError):
            attend(**kw)
    with pytest.raises(ValueError):
        ops.kv_copy_pages(c, ints, ints)
    with pytest.raises(ValueError):
        ops.kv_copy_pages(c, ints, ints[:2])


# ---- pages -----------------------------------------------------------------------
@pytest.fixture
def pool(monkeypatch):
    def copy(cache, src, dst, stream=None):
        assert not set(src.tolist()) & set(dst.tolist()) and len(set(dst.tolist())) == dst.numel()
        for t in (cache.k, cache.v):
            t[:, dst.long()] = t[:, src.long()]

    monkeypatch.setattr(ops, "kv_copy_pages", copy)

    def make(**kw):
        a = dict(layers=2, pages=12, kv_heads=2, head_dim=8, page_size=4, max_seqs=5, dtype=torch.float32, device="cpu")
        return PagedKvCache(**{**a, **kw})

    return make


class Checked:
    """A PagedKvCache whose slots hold a number for each token, beside plain lists of those numbers."""

    def __init__(self, kv):
        self.kv, self.want, self.next = kv, {}, 1.0

    def extend(self, seqs, counts):
        self.kv.extend(seqs, counts)
        for s, n in zip(seqs, counts):
            for _ in range(n):
                t = len(self.want[s])
                page = int(self.kv.page_table[s, t // self.kv.page_size])
                self.kv.cache.k[:, page, :, t % self.kv.page_size] = self.next
                self.kv.cache.v[:, page, :, t % self.kv.page_size] = -self.next
                self.want[s].append(self.next)
                self.next += 1.0

    def check(self):
        kv, holders = self.kv, {}
        for s, want in self.want.items():
            assert kv.length(s) == len(want) and len(kv.pages(s)) == -(-len(want) // kv.page_size)
            assert kv.page_table[s, :len(kv.pages(s))].tolist() == kv.pages(s)
            assert (kv.page_table[s, len(kv.pages(s)):] == -1).all()
            for t, x in enumerate(want):
                page = kv.pages(s)[t // kv.page_size]
                assert (kv.cache.k[:, page, :, t % kv.page_size] == x).all()
                assert (kv.cache.v[:, page, :, t % kv.page_size] == -x).all()
            for p in kv.pages(s):
                holders[p] = holders.get(p, 0) + 1
        assert kv.free_pages == kv.cache.pages - len(holders)


@pytest.mark.parametrize("layout", ["heads", "tokens"])
def test_forks_share_until_written(pool, layout):
    c = Checked(pool(layout=layout))
    a = c.kv.new()
    c.want[a] = []
    c.extend([a], [6])
    b = c.kv.fork(a)
    c.want[b] = list(c.want[a])
    assert c.kv.pages(a) == c.kv.pages(b) and c.kv.free_pages == 10
    c.extend([a, b], [1, 1])  # one of the two keeps the half-filled page
    c.check()
    assert c.kv.pages(a)[0] == c.kv.pages(b)[0] and c.kv.pages(a)[1] != c.kv.pages(b)[1] and c.kv.free_pages == 9
    c.extend([b], [1])
    d = c.kv.fork(b)  # its last page is full: the fork's next token needs no copy
    c.want[d] = list(c.want[b])
    c.extend([d], [1])
    c.check()
    assert c.kv.pages(d)[:2] == c.kv.pages(b)
    c.kv.free(a)
    del c.want[a]
    c.check()


def test_random_use_keeps_every_token(pool):
    rng = np.random.default_rng(3)
    c = Checked(pool(pages=24, max_seqs=6))
    done = dict.fromkeys(("new", "fork", "free", "compact", "extend", "full"), 0)
    for _ in range(600):
        live = list(c.want)
        what = rng.choice(["new", "fork", "free", "compact", "extend", "extend", "extend"])
        try:
            if what == "new":
                s = c.kv.new()
                c.want[s] = []
            elif what == "fork" and live:
                s = int(rng.choice(live))
                new = c.kv.fork(s)
                c.want[new] = list(c.want[s])
            elif what == "free" and live:
                s = int(rng.choice(live))
                c.kv.free(s)
                del c.want[s]
            elif what == "compact":
                c.kv.compact()
                used = sorted({p for s in c.want for p in c.kv.pages(s)})
                assert used == list(range(len(used)))
            elif what == "extend" and live:
                some = [int(s) for s in rng.permutation(live)[:rng.integers(1, len(live) + 1)]]
                c.extend(some, [int(n) for n in rng.integers(0, 6, len(some))])
            done[what] += 1
        except MemoryError:
            done["full"] += 1
        c.check()
    assert all(done.values())


def test_pages_run_out_without_a_trace(pool):
    c = Checked(pool(pages=3, max_pages=2, max_seqs=3))
    a, b = c.kv.new(), c.kv.new()
    c.want = {a: [], b: []}
    c.extend([a], [5])
    for seqs, counts in (([a, b], [1, 5]), ([a], [4])):
        with pytest.raises(MemoryError):
            c.kv.extend(seqs, counts)
        c.check()
    c.kv.new()
    for call in (c.kv.new, lambda: c.kv.fork(a)):
        with pytest.raises(MemoryError):
            call()
    for args in (([a, a], [1, 1]), ([a], [1, 1]), ([a], [-1])):
        with pytest.raises(ValueError):
            c.kv.extend(*args)
    with pytest.raises(ValueError):
        pool(layout="rows")
    with pytest.raises(ValueError):
        pool(pages=0)
    c.check()


def test_unknown_sequences_are_refused_without_a_trace(pool):
    c = Checked(pool(max_seqs=3))
    a, b = c.kv.new(), c.kv.new()
    c.want = {a: []}
    c.extend([a], [3])
    c.kv.free(b)
    for unknown in (b, 7):  # b's row is the one that a fork would take
        for call in (c.kv.fork, c.kv.free, c.kv.length, c.kv.pages, lambda s: c.kv.extend([a, s])):
            with pytest.raises(KeyError):
                call(unknown)
    c.check()
    for _ in range(2):  # both rows are still to be had
        c.want[c.kv.new()] = []
    c.check()
    with pytest.raises(ValueError):
        pool(max_pages=0)


def test_attention_in_place_takes_one_stride():
    for change in (dict(out_stride=516), dict(q_stride=516), dict(q_stride=1024, rows=2)):
        assert _lib.lib().mli_paged_attention(attention(**change), cache(), 0, None) == INVALID


def test_caches_whose_heads_lie_on_one_another_are_refused():
    l = _lib.lib()
    for change in (dict(slot_stride=0), dict(slot_stride=56), dict(head_stride=0), dict(page_stride=32),
                   dict(layer_stride=0), dict(layers=1, layer_stride=0, page_stride=0)):
        c = cache(**change)
        assert l.mli_rope_append(rope(), c, 0, None) == INVALID
        assert l.mli_paged_attention(attention(), c, 0, None) == INVALID
        assert l.mli_kv_copy_pages(c, A, A, 1, None) == INVALID
    one = torch.zeros(1, 1, 1, 16, 64)
    for n in ((2, 1, 1), (1, 2, 1), (1, 1, 2)):
        t = one.expand(*n, 16, 64)
        with pytest.raises(ValueError, match="memory of its own"):
            ops.KvCache(t, t)
    t = torch.zeros(1, 2, 4, 17 * 32 + 32).as_strided((1, 2, 4, 16, 64), (0, 2304, 576, 32, 1))  # rows of 64, 32 apart
    with pytest.raises(ValueError, match="memory of its own"):
        ops.KvCache(t, t)
    ops.KvCache(one.expand(1, 1, 1, 16, 64), one)  # a stride of 0 over one entry is none


def test_tiles_are_counted_once_for_every_eight_heads():
    """rows * kv_heads * ceil(group / 8) * (tokens / 8) of an fp32 cache of 256 dims, whose tiles are the smallest."""
    c = cache(dtype=0, head_dim=256, layer_stride=8 * 4 * 16 * 256, page_stride=4 * 16 * 256, head_stride=16 * 256,
              slot_stride=256)
    wide = dict(rows=256, q_stride=128 * 256, out_stride=128 * 256, q=2 * A, table_cols=948000, table_stride=948000)
    assert 256 * 4 * (948000 * 16 // 8) < 2e9 < 256 * 4 * 2 * (948000 * 16 // 8)
    for heads in (36, 64, 128):  # groups of 9, 16 and 32: two passes and four
        assert _lib.lib().mli_paged_attention(attention(heads=heads, **wide), c, 0, None) == UNSUPPORTED


@pytest.mark.parametrize("broken", ["copy", "upload"])
def test_device_calls_that_fail_leave_no_trace(pool, monkeypatch, broken):
    """A page copy or an update of the page table that raises (no memory, a capture under way): the sequences, their
    pages and the free ones are what they were, and the same call succeeds later."""
    c = Checked(pool(pages=16))

    def trace():
        kv = c.kv
        return (dict(kv._lengths), {s: list(p) for s, p in kv._pages.items()}, list(kv._holders), list(kv._free_pages),
                list(kv._free_rows), kv.page_table.clone())

    def fails(call, copies=True):
        before = trace()
        with monkeypatch.context() as m:
            def raises(*args, **kw):
                raise RuntimeError("broken")

            if broken == "copy":
                m.setattr(ops, "kv_copy_pages", raises)
            else:
                m.setattr(c.kv, "page_table", _Unwritable(c.kv.page_table))
            if broken == "upload" or copies:
                with pytest.raises(RuntimeError, match="broken"):
                    call()
                assert trace()[:5] == before[:5]
        assert torch.equal(c.kv.page_table, before[5])
        c.check()

    a, b = c.kv.new(), c.kv.new()
    c.want = {a: [], b: []}
    fails(lambda: c.kv.extend([a, b], [6, 9]), copies=False)
    c.extend([a, b], [6, 9])
    fails(lambda: c.kv.fork(a), copies=False)
    d = c.kv.fork(a)
    c.want[d] = list(c.want[a])
    fails(lambda: c.kv.extend([a, d, b], [1, 3, 4]))
    c.extend([a, d, b], [1, 3, 4])
    c.check()
    fails(lambda: c.kv.free(b), copies=False)
    c.kv.free(a)
    del c.want[a]
    fails(c.kv.compact)
    assert c.kv.compact() > 0
    c.check()


class _Unwritable:
    """A page table that can be read, and whose every write raises."""

    def __init__(self, table):
        self._table, self.device = table, table.device

    def clone(self):
        return self._table.clone()

    def __getitem__(self, at):
        return self

    def __setitem__(self, at, value):
        raise RuntimeError("broken")

    def fill_(self, value):
        raise RuntimeError("broken")


@pytest.mark.parametrize("seqs", [1, 2, 7])
def test_only_entries_that_change_are_written(pool, monkeypatch, seqs):
    """A token in a new page writes its one entry, a copied page its one; a compaction those of the pages it moved."""
    c = Checked(pool(pages=200, max_seqs=9))
    sent, write = [], c.kv._write
    monkeypatch.setattr(c.kv, "_write", lambda *lists: (sent.append([list(x) for x in lists]), write(*lists))[1])
    all_, b = [c.kv.new() for _ in range(seqs)], c.kv.new()
    c.want = {s: [] for s in [*all_, b]}
    c.extend([b], [7])
    c.extend(all_, [76] * seqs)
    sent.clear()
    c.extend([*all_, b], [1] * seqs + [1])
    assert sent == [[all_, [19] * seqs, [c.kv.pages(s)[19] for s in all_]]]
    sent.clear()
    c.extend([*all_, b], [1] * seqs + [0])
    assert not sent
    d = c.kv.fork(all_[0])
    c.want[d] = list(c.want[all_[0]])
    c.extend([d], [1])
    assert sent == [[[d], [19], [c.kv.pages(d)[19]]]]
    c.kv.free(b)
    del c.want[b]
    sent.clear()
    before = {s: c.kv.pages(s) for s in [*all_, d]}
    assert c.kv.compact() == 2
    changed = [(s, i, p) for s in before for i, p in enumerate(c.kv.pages(s)) if p != before[s][i]]
    assert sorted(zip(*sent[0])) == sorted(changed)
    c.check()
