"""Decode steps that queue the paged cache's operators back to back with one another and with chained GEMVs, on a
stream whose launches may overlap (programmatic dependent launch), eagerly and replayed from a captured graph.  The same
calls one at a time, without overlap, give the bits to hold them against; those are checked against the formulas."""
import math

import numpy as np
import pytest

from minillama_infra_b200 import ops, synth
from oracle import oracle as orc
from test_kv_cache_gpu import BF16, F32, check_rope, check_row, empty_cache, gen, i32, normal

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def on_stream(stream, call):
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
    torch.cuda.current_stream().wait_stream(stream)


def captured(stream, call):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call()
    return graph


class Layers:
    """Four layers of calls that share one workspace, one buffer of rotated queries and one of outputs: an append, a copy
    of the pages it wrote, attention over the copies, an append of the outputs to a cache that logs them, another
    attention of other lengths, and its log.  Every layer has its own inputs, lengths and pages."""

    heads, group, dim, page, layers = 2, 4, 64, 16, 4
    lengths = ([9000, 40, 0, 2000], [17, 9000, 300, 1], [0, 1, 5000, 8999], [64, 0, 4097, 9000])
    others = ([3, 700, 1, 33], [8000, 0, 2, 299], [1, 1, 4000, 16], [63, 0, 4000, 1])

    def __init__(self, g, dtype):
        m, h, hq = 4, self.heads, self.heads * self.group
        per = -(-9000 // self.page)
        spare = m * self.layers
        self.c = empty_cache(self.layers, m * per + spare, h, self.page, self.dim, dtype)
        self.log = empty_cache(2 * self.layers, m, hq, 1, self.dim, F32, fill=0.0)
        self.start = [normal(g, *self.c.k.shape).to(dtype) for _ in range(2)]
        self.table = torch.randperm(m * per, generator=g, device="cuda").to(torch.int32).view(m, per)
        self.copies, self.pos, self.lens, self.short = [], [], [], []
        for i in range(self.layers):
            src, dst, table = [], [], self.table.clone()
            for r, n in enumerate(self.lengths[i]):
                col, free = max(0, n - 1) // self.page, m * per + i * m + r
                src.append(int(table[r, col]) if n else -1)
                dst.append(free)
                if n:
                    table[r, col] = free
            self.copies.append((i32(src), i32(dst), table))
            self.pos.append(i32([n - 1 for n in self.lengths[i]]))
            self.lens.append(i32(self.lengths[i]))
            self.short.append(i32(self.others[i]))
        self.qs = [normal(g, m, hq, self.dim) for _ in range(self.layers)]
        self.ks, self.vs = ([normal(g, m, h, self.dim) for _ in range(self.layers)] for _ in range(2))
        self.q, self.out, self.unused = (torch.empty_like(self.qs[0]) for _ in range(3))
        self.turns = ops.rope_turns(self.dim)
        self.ws = ops.paged_attention_workspace(self.c, m, hq)
        self.zeros, self.log_table = i32([0] * m), torch.arange(m, device="cuda", dtype=torch.int32)[:, None].contiguous()

    def reset(self):
        self.c.k.copy_(self.start[0])
        self.c.v.copy_(self.start[1])
        for t in (self.log.k, self.log.v, self.out):
            t.fill_(math.nan)
        self.q.zero_()

    def run(self, between=lambda: None):
        def note(where):  # the outputs, as values of a token of every row
            ops.rope_append(self.unused, self.out, self.out, self.out, self.log, where, self.zeros, self.log_table, None)
            between()

        for i in range(self.layers):
            src, dst, table = self.copies[i]
            ops.rope_append(self.q, self.qs[i], self.ks[i], self.vs[i], self.c, i, self.pos[i], self.table, self.turns)
            between()
            ops.kv_copy_pages(self.c, src, dst)
            between()
            ops.paged_attention(self.out, self.q, self.c, i, table, self.lens[i], 0.125, self.ws)
            between()
            note(2 * i)
            ops.paged_attention(self.out, self.q, self.c, i, self.table, self.short[i], 0.125, self.ws)
            between()
            note(2 * i + 1)

    def state(self):
        torch.cuda.synchronize()
        return [t.clone() for t in (self.c.k, self.c.v, self.log.k, self.log.v)]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_overlapping_launches_see_what_came_before(dtype):
    g = gen(40)
    d = Layers(g, dtype)
    kept = ops.lib().mli_get_launch_flags()
    ops.set_pdl(False)
    try:
        d.reset()
        d.run(torch.cuda.synchronize)
        want = d.state()
    finally:
        ops.lib().mli_set_launch_flags(kept)
    for i in range(d.layers):
        live = [r for r, n in enumerate(d.lengths[i]) if n]
        for lengths, table, where in ((d.lengths[i], d.copies[i][2], 2 * i), (d.others[i], d.table, 2 * i + 1)):
            for r, n in enumerate(lengths):
                p = table[r].long()
                k, v = (x[i, p].transpose(1, 2).reshape(-1, d.heads, d.dim)[:n] for x in (d.c.k, d.c.v))
                if r in live:  # (queries of padded tokens are those of the layer before)
                    q = rotated(d, i, r)
                    check_row(d.log.v[where, r, :, 0], q, k, v, 0.125, f"layer {i}, row {r}")
    ops.set_pdl(True)
    stream = torch.cuda.Stream()
    try:
        for _ in range(5):
            d.reset()
            on_stream(stream, d.run)
            assert all(same(a, b) for a, b in zip(d.state(), want))
        graph = captured(stream, d.run)
        for _ in range(5):
            d.reset()
            on_stream(stream, graph.replay)
            assert all(same(a, b) for a, b in zip(d.state(), want))
    finally:
        ops.lib().mli_set_launch_flags(kept)
    assert ops.device_error() == 0


def rotated(d, layer, row):
    """The rotated queries of one row, by a call of their own."""
    q, c = torch.empty_like(d.q), empty_cache(1, 1, d.heads, 1, d.dim, F32)
    ops.rope_append(q, d.qs[layer], d.ks[layer], d.vs[layer], c, 0, d.pos[layer], torch.full_like(d.table, -1), d.turns)
    assert ops.device_error() == 6  # queries only
    check_rope(q[row:row + 1], d.qs[layer][row:row + 1], d.pos[layer][row:row + 1].long(), d.turns, False, None)
    return q[row]


class Decoder:
    """Layers of the 1B model's sizes, batch 1: the linear layers, norms, SwiGLU and residuals in chained launches, the
    rotation, append and attention between them."""

    dim, hidden, heads, kv_heads, head = 2048, 8192, 32, 8, 64

    def __init__(self, g, form, dtype, layers):
        self.form, self.layers, kv = form, layers, self.kv_heads * self.head
        rows = ((self.dim, self.dim), (kv, self.dim), (kv, self.dim), (self.dim, self.dim), (self.hidden, self.dim),
                (self.hidden, self.dim), (self.dim, self.hidden))
        self.w = [[synth.weights_gpu(d, n, seed=100 * i + j, device=torch.device("cuda:0"))
                   for j, (d, n) in enumerate(rows)] for i in range(layers)]
        self.norms = [[1 + 0.1 * normal(g, self.dim) for _ in range(2)] for _ in range(layers)]
        sizes = dict(q=(1, self.heads, self.head), k=(1, self.kv_heads, self.head), v=(1, self.kv_heads, self.head),
                     rotated=(1, self.heads, self.head), att=(self.dim,), h=(self.hidden,))
        self.b = [{name: torch.empty(size, device="cuda") for name, size in sizes.items()} for _ in range(layers)]
        self.x, self.start = torch.empty(self.dim, device="cuda"), torch.empty(self.dim, device="cuda")
        self.chains = [ops.GemvChain(self.project(0, 0))]
        for i in range(layers):
            self.chains.append(ops.GemvChain(self.rest(i) + (self.project(i + 1, 4) if i + 1 < layers else [])))
        self.c = empty_cache(layers, 40, self.kv_heads, 16, self.head, dtype, fill=0.0)
        self.table = torch.randperm(40, generator=g, device="cuda").to(torch.int32)[None]
        self.turns = ops.rope_turns(self.head, scaling="llama3", factor=32.0)
        self.ws = ops.paged_attention_workspace(self.c, 1, self.heads)
        self.pos, self.length = i32([0]), i32([1])

    def op(self, i, j, wait, **kw):
        d, n = self.w[i][j][0].shape
        return dict(form=self.form, n=n, d=d, wait=wait, w_q=self.w[i][j][0], w_s=self.w[i][j][1], **kw)

    def project(self, i, wait):
        return [self.op(i, j, wait, x=self.x, norm_w=self.norms[i][0], y=self.b[i][name])
                for j, name in enumerate("qkv")]

    def rest(self, i):
        b, norm = self.b[i], self.norms[i][1]
        return [self.op(i, 3, 0, x=b["att"], y=self.x, epilogue="add"),
                self.op(i, 4, 1, x=self.x, norm_w=norm, y=b["h"], epilogue="swiglu"),
                self.op(i, 5, 1, x=self.x, norm_w=norm, y=None),
                self.op(i, 6, 3, x=b["h"], y=self.x, epilogue="add")]

    def step(self):
        self.x.copy_(self.start)
        self.chains[0].run()
        for i, b in enumerate(self.b):
            ops.rope_append(b["rotated"], b["q"], b["k"], b["v"], self.c, i, self.pos, self.table, self.turns)
            ops.paged_attention(b["att"].view(1, self.heads, self.head), b["rotated"], self.c, i, self.table, self.length,
                                0.125, self.ws)
            self.chains[i + 1].run()

    def single(self, x, i, j):
        d, n = self.w[i][j][0].shape
        y, x = torch.empty(d, device="cuda"), torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda()
        (ops.matmul_int8 if self.form == "w8a32" else ops.matmul_dp4a_fused)(y, x, *self.w[i][j], n, d, 64)
        return y.cpu().numpy()

    def check(self):
        """Every operator of the last step against its own inputs."""
        n, exp = int(self.length), self.start.cpu().numpy().copy()
        p = self.table[0].long()
        for i, b in enumerate(self.b):
            xa = orc.rmsnorm_chain(exp, self.norms[i][0].cpu().numpy())
            for j, name in enumerate("qkv"):
                assert np.array_equal(b[name].cpu().numpy().ravel().view(np.uint32), self.single(xa, i, j).view(np.uint32))
            check_rope(b["rotated"], b["q"], self.pos.long(), self.turns, False, None)
            k, v = (t[i, p].transpose(1, 2).reshape(-1, self.kv_heads, self.head)[:n] for t in (self.c.k, self.c.v))
            check_rope(k[-1:], b["k"], self.pos.long(), self.turns, False, None)
            assert torch.equal(v[-1], b["v"][0].to(v.dtype))
            check_row(b["att"].view(self.heads, self.head), b["rotated"][0], k, v, 0.125, f"layer {i}, {n} tokens")
            exp = (exp + self.single(b["att"].cpu().numpy(), i, 3)).astype(np.float32)
            xf = orc.rmsnorm_chain(exp, self.norms[i][1].cpu().numpy())
            gate, up = (torch.from_numpy(self.single(xf, i, j)) for j in (4, 5))
            h, want = b["h"].cpu().numpy(), (gate * (1.0 / (1.0 + torch.exp(-gate))) * up).numpy()
            assert orc.max_abs_rel(h, want) <= 1e-6
            exp = (exp + self.single(h, i, 6)).astype(np.float32)
        assert np.array_equal(self.x.cpu().numpy().view(np.uint32), exp.view(np.uint32))


@pytest.mark.parametrize("form,dtype", [("w8a32", BF16), ("w8a8_fused", F32)])
def test_layers_of_chains_appends_and_attention(form, dtype):
    """Tokens decoded one after another through a stack of layers, each step queued without a wait on a stream of its own:
    every operator's output is right for its inputs, and a captured step replayed over the same tokens gives the same
    bits of every one."""
    g = gen(41)
    d = Decoder(g, form, dtype, 3)
    prompt = [normal(g, *d.c.k.shape).to(dtype) for _ in range(2)]
    xs = [normal(g, d.dim) for _ in range(4)]
    stream = torch.cuda.Stream()

    def decode(step, check):
        seen = []
        d.c.k.copy_(prompt[0])
        d.c.v.copy_(prompt[1])
        for t, x in enumerate(xs):
            d.start.copy_(x)
            d.pos.fill_(600 + t)  # on to the 38th page
            d.length.fill_(601 + t)
            on_stream(stream, step)
            torch.cuda.synchronize()
            seen.append([d.x.clone()] + [t.clone() for b in d.b for t in b.values()])
            if check:
                d.check()
        return seen + [[d.c.k.clone(), d.c.v.clone()]]

    want = decode(d.step, True)
    graph = captured(stream, d.step)
    got = decode(graph.replay, False)
    for a, b in zip(got, want):
        assert all(same(x, y) for x, y in zip(a, b))
    assert ops.device_error() == 0
    del graph
    for c in d.chains:
        c.close()
