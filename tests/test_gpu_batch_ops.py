"""The operators of a batched step on the device against plain 64-bit forms (batch_ops_ref): row norms,
cache pages, the append, attention over the pages, low-rank adapters, and a step of all of them.

Tolerances count roundings: a value of a type is off by at most half a step, eps / 2 of it."""
import numpy as np
import pytest
import torch

import batch_ops_ref as R
from charsiu_b200 import gguf as G
from charsiu_b200 import workloads as W
from charsiu_b200.lib import AdaptersStruct, AttentionStruct, GpuError, Layer, PagesStruct
from oracle import oracle as O

pytestmark = pytest.mark.gpu

F16, BF16 = 1, 30
TYPES = {F16: torch.float16, BF16: torch.bfloat16}
EPS = {F16: 2.0 ** -10, BF16: 2.0 ** -7}


@pytest.fixture(scope="module")
def layer():
    with Layer(2048, 2048, 8) as g:
        yield g


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(dtype)).cuda()


def st():
    return torch.cuda.current_stream().cuda_stream or 1


def scratch(n):
    return torch.zeros(max(n, 16), dtype=torch.uint8, device="cuda")


# ---- the norm --------------------------------------------------------------------


def run_norm(g, x, add, w, eps=1e-5, out="new"):
    m, k = x.shape
    q = torch.full((m + 1, k), 77, dtype=torch.int8, device="cuda")
    d = torch.full((m + 1, k // 32), 77.0, device="cuda")
    xo = {"new": torch.empty(m, k, device="cuda"), "x": x, "add": add, None: None}[out]
    g.norm_quantise_dev(x.data_ptr(), add.data_ptr() if add is not None else 0, w.data_ptr(), m, k, eps,
                        xo.data_ptr() if xo is not None else 0, q.data_ptr(), d.data_ptr(), st())
    torch.cuda.synchronize()
    assert (q[m] == 77).all() and (d[m] == 77).all()
    return xo, q[:m], d[:m]


@pytest.mark.parametrize("m,k", [(1, 32), (1, 2048), (2, 64), (3, 96), (5, 2016), (7, 4096), (1, 8192),
                                 (33, 1024), (150, 8160), (1000, 256), (640, 2048)])
@pytest.mark.parametrize("residual", [True, False])
def test_norm_is_the_decode_steps(layer, m, k, residual):
    rng = np.random.default_rng(m * 8192 + k)
    x = rng.standard_normal((m, k)).astype(np.float32) * 10.0 ** rng.uniform(-3, 3, (m, 1)).astype(np.float32)
    add = rng.standard_normal((m, k)).astype(np.float32) if residual else None
    w = (1 + 0.1 * rng.standard_normal(k)).astype(np.float32)
    s, q, d = R.norm_rows(x, add, w, 1e-5)
    for out in ("new", "x", "add", None) if residual else ("new", None):
        gs, gq, gd = run_norm(layer, dev(x), dev(add) if residual else None, dev(w), out=out)
        assert np.array_equal(gq.cpu().numpy(), q)
        assert np.array_equal(gd.cpu().numpy().view(np.uint32), d.view(np.uint32))
        if gs is not None:
            assert np.array_equal(gs.cpu().numpy().view(np.uint32), s.view(np.uint32))


def test_norm_of_odd_rows(layer):
    """Zero rows, huge and tiny values, inf and NaN beside ordinary rows: a row is its own."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((9, 512)).astype(np.float32)
    x[0] = 0
    x[2] *= 1e18                     # squares stay finite
    x[3] *= 1e-22                    # squares are subnormal or 0
    x[5, 100] = np.inf
    x[6, 511] = np.nan
    x[7] = 0
    x[7, 3] = 1
    w = np.ones(512, np.float32)
    with np.errstate(all="ignore"):
        _, q, d = R.norm_rows(x, None, w, 1e-5)
    _, gq, gd = run_norm(layer, dev(x), None, dev(w), out=None)
    rows = [0, 1, 2, 3, 4, 7, 8]
    assert np.array_equal(gq.cpu().numpy()[rows], q[rows])
    assert np.array_equal(gd.cpu().numpy()[rows].view(np.uint32), d[rows].view(np.uint32))


def test_norm_refusals(layer):
    x, w = torch.zeros(2, 64, device="cuda"), torch.ones(64, device="cuda")
    q, d = torch.zeros(2, 64, dtype=torch.int8, device="cuda"), torch.zeros(2, 2, device="cuda")
    ok = [x.data_ptr(), 0, w.data_ptr(), 2, 64, 1e-5, 0, q.data_ptr(), d.data_ptr(), st()]
    layer.norm_quantise_dev(*ok)
    for at, bad in ((0, 0), (0, ok[0] + 4), (1, ok[0] + 8), (2, 0), (2, ok[2] + 4), (4, 48), (4, 0),
                    (4, 8224), (6, ok[0] + 4), (7, ok[7] + 1), (8, 0), (8, ok[8] + 1)):
        args = list(ok)
        args[at] = bad
        with pytest.raises(GpuError):
            layer.norm_quantise_dev(*args)
    args = list(ok)
    args[3] = 0                       # no rows: nothing to do
    layer.norm_quantise_dev(*args)


# ---- the pages --------------------------------------------------------------------


class Cache:
    """A paged cache on the device with its plain twin."""

    def __init__(self, g, rng, n_seq, max_pages, n_pages, page=16, kv=2, hd=64, layers=2, ty=BF16,
                 layout="phd"):
        self.g, self.page, self.layout = g, page, layout
        if layout == "gaps":              # strides with room between positions, heads and pages
            full = (layers, n_pages + 1, page, kv, 2, hd)
        else:
            full = (layers, n_pages, page, kv, hd) if layout == "phd" else (layers, n_pages, kv, page, hd)
        self.full = [torch.from_numpy(rng.standard_normal(full).astype(np.float32)).to(TYPES[ty]).cuda()
                     for _ in range(2)]
        self.k, self.v = [t[:, :n_pages, :, :, 0] if layout == "gaps" else t if layout == "phd" else
                          t.transpose(2, 3) for t in self.full]
        self.table = torch.full((n_seq, max_pages), 12345, dtype=torch.int32, device="cuda")
        self.len = torch.zeros(n_seq, dtype=torch.int32, device="cuda")
        self.ref = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        s = self.k.stride()
        self.p = PagesStruct(k=self.k.data_ptr(), v=self.v.data_ptr(), table=self.table.data_ptr(),
                             len=self.len.data_ptr(), ref=self.ref.data_ptr(), layer_stride=s[0],
                             page_stride=s[1], pos_stride=s[2], head_stride=s[3], type=ty,
                             n_layer=layers, n_pages=n_pages, page=page, n_head_kv=kv, head_dim=hd,
                             n_seq=n_seq, max_pages=max_pages)
        self.work = scratch(g.pages_work(self.p))
        self.p.work = self.work.data_ptr()

    def plain(self):
        f = lambda t: t.float().cpu().numpy()  # noqa: E731
        return R.Pages(self.table.cpu().numpy(), self.len.cpu().numpy(), self.ref.cpu().numpy(),
                       f(self.k), f(self.v), self.page)

    def same(self, twin, refused0=0):
        torch.cuda.synchronize()
        assert np.array_equal(self.len.cpu().numpy(), twin.len)
        assert np.array_equal(self.ref.cpu().numpy(), twin.ref)
        assert np.array_equal(self.table.cpu().numpy(), twin.table)
        assert self.refused() - refused0 == twin.refused
        for got, want in ((self.k, twin.k), (self.v, twin.v)):
            assert np.array_equal(got.float().cpu().numpy(), want)

    def refused(self):
        return int(self.work[:4].view(torch.int32)[0])

    def ints(self, v):
        return torch.tensor(list(v), dtype=torch.int32, device="cuda")

    def grow(self, slots, add):
        s = self.ints(slots)
        self.g.pages_grow_dev(self.p, s.data_ptr(), len(slots), add, st())

    def fork(self, src, dst):
        a, b = self.ints(src), self.ints(dst)
        self.g.pages_fork_dev(self.p, a.data_ptr(), b.data_ptr(), len(src), st())

    def free(self, slots):
        s = self.ints(slots)
        self.g.pages_free_dev(self.p, s.data_ptr(), len(slots), st())

    def compact(self):
        live = torch.full((1,), -1, dtype=torch.int32, device="cuda")
        self.g.pages_compact_dev(self.p, live.data_ptr(), st())
        return int(live)


LAYOUTS = ["phd", "hpd", "gaps"]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("page,ty,hd", [(16, BF16, 64), (32, F16, 128), (128, BF16, 64)])
def test_pages_at_random(layer, layout, page, ty, hd):
    """Grows, forks, frees and packings in a random order, refusals among them (slots out of range or
    listed twice, forks into used slots, tables and pools that run out): the plain steps' state, and
    nothing else is written (unused table entries and pages, the gaps between)."""
    rng = np.random.default_rng(page + hd + len(layout))
    c = Cache(layer, rng, n_seq=12, max_pages=6, n_pages=37, page=page, ty=ty, hd=hd, layout=layout)
    other = [t.clone() for t in c.full]
    twin = c.plain()
    for step in range(60):
        what, n = rng.integers(4), int(rng.integers(1, 8))
        a, b = rng.integers(-1, 13, size=n).tolist(), rng.integers(-1, 13, size=n).tolist()
        if what == 0:
            add = int(rng.choice([1, page - 1, page, 3 * page + 5]))
            c.grow(a, add)
            twin.grow(a, add)
        elif what == 1:
            c.fork(a, b)
            twin.fork(a, b)
        elif what == 2:
            c.free(a[:3])
            twin.free(a[:3])
        elif step % 3 == 0:
            assert c.compact() == twin.compact()
        c.same(twin)
    assert twin.refused > 20
    if layout == "gaps":
        for got, was in zip(c.full, other):
            assert torch.equal(got[:, :, :, :, 1], was[:, :, :, :, 1])
            assert torch.equal(got[:, 37], was[:, 37])


def test_pages_many_items(layer):
    """As many slots as a call takes, more pages than one pass of the scan, a pool that runs out."""
    rng = np.random.default_rng(8)
    c = Cache(layer, rng, n_seq=2100, max_pages=5, n_pages=9001, kv=1, layers=1)
    twin = c.plain()
    a = rng.permutation(2100)[:1024].tolist()
    for add in (1, 40):
        c.grow(a, add)
        twin.grow(a, add)
    c.same(twin)
    b = [s for s in range(2100) if s not in set(a)][:1024]
    for obj in (c, twin):
        obj.free(a[::3])
        obj.fork([a[i] for i in range(1024)], b)
    c.same(twin)
    for obj in (c, twin):
        obj.grow(b, 30)
        obj.grow(a, 33)
        obj.free(b[::2])
        obj.grow(a, 17)
    c.same(twin)
    assert c.compact() == twin.compact()
    c.same(twin)


def test_pages_growth_past_every_pool(layer):
    """Growths past 31 bits of positions or past the table are refused, nothing else."""
    c = Cache(layer, np.random.default_rng(0), n_seq=3, max_pages=4, n_pages=5, kv=1, layers=1)
    twin = c.plain()
    for obj in (c, twin):
        obj.grow([0, 1, 2], 0x7fffffff)
        obj.grow([0, 1, 2], 16)
        obj.grow([0, 1, 2], 32)
    c.same(twin)


def test_pages_growths_whose_needs_pass_32_bits(layer):
    """64 slots that ask for 2^26 pages each, of a pool of 5: the needs add up to 2^32, and all are
    refused. (The table is as large as told; nothing of it is touched.)"""
    c = Cache(layer, np.random.default_rng(0), n_seq=64, max_pages=4, n_pages=5, kv=1, layers=1)
    wide = 1 << 26
    table = torch.empty(64 * wide, dtype=torch.int32, device="cuda")
    c.p.table, c.p.max_pages = table.data_ptr(), wide
    c.grow(range(64), wide * 16)
    assert c.refused() == 64 and not c.len.any() and not c.ref.any()
    c.grow([3, 1], 30)
    assert c.refused() == 64 and c.len.tolist()[:4] == [0, 30, 0, 30] and c.ref.tolist() == [1, 1, 1, 1, 0]
    assert table[3 * wide:3 * wide + 2].tolist() == [0, 1] and table[wide:wide + 2].tolist() == [2, 3]


def test_pages_calls_that_do_nothing(layer):
    c = Cache(layer, np.random.default_rng(1), n_seq=3, max_pages=4, n_pages=5)
    twin = c.plain()
    s = c.ints([0])
    layer.pages_grow_dev(c.p, s.data_ptr(), 0, 1, st())
    layer.pages_grow_dev(c.p, s.data_ptr(), 1, 0, st())
    layer.pages_fork_dev(c.p, s.data_ptr(), s.data_ptr(), 0, st())
    layer.pages_free_dev(c.p, s.data_ptr(), 0, st())
    c.fork([0, 1], [1, 0])                 # empty sources: empty forks
    twin.fork([0, 1], [1, 0])
    c.free([2, 2])
    assert c.compact() == 0
    c.same(twin)


def test_pages_refusals(layer):
    c = Cache(layer, np.random.default_rng(1), n_seq=3, max_pages=4, n_pages=5)
    s = c.ints([0, 1])
    with pytest.raises(GpuError):
        layer.pages_grow_dev(c.p, 0, 1, 1, st())
    with pytest.raises(GpuError):
        layer.pages_grow_dev(c.p, s.data_ptr(), 1025, 1, st())
    with pytest.raises(GpuError):
        layer.pages_grow_dev(c.p, s.data_ptr(), 1, 0x80000000, st())
    with pytest.raises(GpuError):
        layer.pages_fork_dev(c.p, s.data_ptr(), 0, 1, st())
    with pytest.raises(GpuError):
        layer.pages_compact_dev(c.p, 2, st())
    c.p.work = None
    with pytest.raises(GpuError):
        layer.pages_free_dev(c.p, s.data_ptr(), 1, st())
    c.p.work = c.work.data_ptr()
    c.p.page = 20
    with pytest.raises(GpuError):
        layer.pages_free_dev(c.p, s.data_ptr(), 1, st())


def test_pages_lists_that_are_misaligned(layer):
    """A list of slots at an odd address is refused on the host (the planners read whole words)."""
    c = Cache(layer, np.random.default_rng(1), n_seq=3, max_pages=4, n_pages=5)
    s = c.ints([0, 1, 2])
    for off in (1, 2, 3):
        bad = s.data_ptr() + off
        with pytest.raises(GpuError):
            layer.pages_grow_dev(c.p, bad, 1, 1, st())
        with pytest.raises(GpuError):
            layer.pages_free_dev(c.p, bad, 1, st())
        for src, dst in ((bad, s.data_ptr()), (s.data_ptr(), bad)):
            with pytest.raises(GpuError):
                layer.pages_fork_dev(c.p, src, dst, 1, st())
    layer.pages_grow_dev(c.p, s.data_ptr() + 4, 2, 1, st())
    torch.cuda.synchronize()
    assert c.len.tolist() == [0, 1, 1]


# ---- the append --------------------------------------------------------------------


def rope_table(n_ctx, hd):
    at = np.arange(n_ctx)[:, None] * 10000.0 ** (-np.arange(0, hd, 2) / hd)[None]
    return np.stack((np.cos(at), np.sin(at)), -1).reshape(n_ctx, hd).astype(np.float32)


def turn32(x, cs):
    """RoPE with every product and sum rounded to fp32."""
    p, c = x.reshape(*x.shape[:-1], -1, 2), cs.reshape(*cs.shape[:-1], -1, 2)
    x0, x1, co, si = p[..., 0], p[..., 1], c[..., 0], c[..., 1]
    return np.stack(((x0 * co) - (x1 * si), (x0 * si) + (x1 * co)), -1).reshape(x.shape).astype(np.float32)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("n,t,heads,kv,hd,page,ty", [
    (1, 1, 2, 1, 64, 16, BF16), (5, 1, 8, 2, 64, 16, F16), (3, 7, 6, 2, 128, 32, BF16),
    (2, 70, 4, 4, 64, 64, F16)])
def test_append(layer, layout, n, t, heads, kv, hd, page, ty):
    """Rows go to their positions rounded once, q too; padded slots, positions before the start, behind
    the rope table or on a bad page write nothing."""
    rng = np.random.default_rng(n * t + heads)
    n_ctx = 3 * page
    c = Cache(layer, rng, n_seq=n + 3, max_pages=4, n_pages=4 * (n + 3), page=page, kv=kv, hd=hd,
              layers=3, ty=ty, layout=layout)
    for s in range(n + 3):
        c.grow([s], int(rng.integers(1, n_ctx + 1)))
    c.grow([n], 4 * page)                                 # (refused unless it fits)
    lens = c.len.cpu().numpy()
    table = c.table.cpu().numpy()
    table[n + 1, 0] = 99999
    c.table.copy_(torch.from_numpy(table))
    slots = [s for s in range(n + 3)] + [-1, n + 3]
    rows = len(slots) * t
    q, k, v = (rng.standard_normal((rows, h, hd)).astype(np.float32) for h in (heads, kv, kv))
    cs = rope_table(n_ctx, hd)
    want = c.plain()
    dt = TYPES[ty]
    q_out = torch.full((rows, heads, hd), 3.0, dtype=dt, device="cuda")
    q_want = q_out.clone()
    layer_at = 1
    to = lambda a: torch.from_numpy(a).to(dt).float().numpy()  # noqa: E731
    for i, s in enumerate(slots):
        for j in range(t):
            if not 0 <= s < n + 3:
                continue
            pos = int(lens[s]) - t + j
            if pos < 0 or pos >= n_ctx or not 0 <= table[s, pos // page] < 4 * (n + 3):
                continue
            r = i * t + j
            q_want[r] = torch.from_numpy(turn32(q[r], cs[pos])).to(dt)
            want.k[layer_at, table[s, pos // page], pos % page] = to(turn32(k[r], cs[pos]))
            want.v[layer_at, table[s, pos // page], pos % page] = to(v[r])
    a = [dev(x) for x in (q, k, v, cs)]
    sl = c.ints(slots)
    layer.pages_append_dev(c.p, layer_at, sl.data_ptr(), len(slots), t, heads, a[0].data_ptr(),
                           a[1].data_ptr(), a[2].data_ptr(), a[3].data_ptr(), n_ctx, q_out.data_ptr(), st())
    torch.cuda.synchronize()
    assert torch.equal(q_out, q_want)
    assert np.array_equal(c.k.float().cpu().numpy(), want.k)
    assert np.array_equal(c.v.float().cpu().numpy(), want.v)


def test_append_refusals(layer):
    c = Cache(layer, np.random.default_rng(1), n_seq=3, max_pages=4, n_pages=5)
    buf = torch.zeros(4096, device="cuda")
    s = c.ints([0, 1])
    p = buf.data_ptr()
    ok = [c.p, 0, s.data_ptr(), 2, 1, 4, p, p, p, p, 8, p, st()]
    layer.pages_append_dev(*ok)                          # empty slots: writes nothing
    for at, bad in ((1, 2), (2, 0), (5, 0), (5, 3), (6, 0), (6, p + 4), (7, p + 8), (8, 0), (9, p + 4), (11, p + 2)):
        args = list(ok)
        args[at] = bad
        with pytest.raises(GpuError):
            layer.pages_append_dev(*args)
    for at in (3, 4):
        args = list(ok)
        args[at] = 0
        layer.pages_append_dev(*args)


# ---- attention -----------------------------------------------------------------------


def build_batch(g, rng, sizes, shared, t, heads, kv, hd, page, ty, layout="phd", layers=2, at=1, spare=3,
                pad=0):
    """Sequences of these own lengths in groups that share `shared` pages each: (cache, slots, group
    bounds, shared pages). sizes: a list a group."""
    n = sum(len(s) for s in sizes)
    longest = max(sh * page + max(s, default=0) for sh, s in zip(shared, sizes))
    max_pages = max(1, -(-longest // page))
    need = sum(shared) + sum(-(-x // page) for s in sizes for x in s) + spare
    c = Cache(g, rng, n_seq=n + 2, max_pages=max_pages, n_pages=need, page=page, kv=kv, hd=hd, ty=ty,
              layout=layout, layers=layers)
    order = rng.permutation(need).tolist()
    table = np.full((n + 2, max_pages), -7, np.int32)
    lens = np.zeros(n + 2, np.int32)
    slots = rng.permutation(n + 2)[:n]
    i = 0
    bounds = [0]
    for sh, s in zip(shared, sizes):
        common = [order.pop() for _ in range(sh)]
        for own in s:
            mine = common + [order.pop() for _ in range(-(-own // page))]
            table[slots[i], :len(mine)] = mine
            lens[slots[i]] = sh * page + own
            i += 1
        bounds.append(i)
    c.table.copy_(torch.from_numpy(table))
    c.len.copy_(torch.from_numpy(lens))
    return c, slots.tolist() + [-1] * pad, bounds, lens, table


def run_attention(g, c, slots, bounds, shared, t, heads, q, at=1, out_type=None, max_len=None, groups=True,
                  scale=None):
    hd = c.k.shape[-1]
    n = len(slots)
    ty = int(c.p.type) if out_type is None else out_type
    out = torch.full((n * t + 1, heads, hd), 55.0, dtype=torch.float32 if ty == 0 else TYPES[ty], device="cuda")
    sl, gr, sh = c.ints(slots), c.ints(bounds), c.ints(shared)
    b = AttentionStruct(slots=sl.data_ptr(), group=gr.data_ptr() if groups else None,
                        shared=sh.data_ptr() if groups else None, n_seq=n, n_tok=t, n_head=heads,
                        n_group=len(shared) if groups else 0,
                        max_len=int(c.len.max()) if max_len is None else max_len, out_type=ty,
                        scale=hd ** -0.5 if scale is None else scale)
    w = torch.full((g.attention_work(c.p, b) + 16,), 255, dtype=torch.uint8, device="cuda")
    b.work, b.work_bytes = w.data_ptr(), w.numel() - 16
    g.attention_dev(c.p, at, b, q.data_ptr(), out.data_ptr(), st())
    torch.cuda.synchronize()
    assert (w[-16:] == 255).all() and (out[n * t:] == 55).all()
    return out[:n * t]


def check_attention(c, slots, lens, table, t, heads, q, out, at=1, scale=None):
    """Against 64 bits. Of the bound: the weights' rounding to the cache's type (half a step of a weight,
    2^-25 where fp16's are subnormal), the scores' (hd + 3 roundings of a sum of |q k|, twice: in the
    weight and in the sum), 2^-20 for exp2 and the joins, half a step of the result."""
    hd, page, ty = c.k.shape[-1], c.page, int(c.p.type)
    scale = hd ** -0.5 if scale is None else scale
    kk, vv = (x[at].double().cpu().numpy() for x in (c.k, c.v))
    qq, got = q.double().cpu().numpy().reshape(len(slots), t, heads, hd), out.double().cpu().numpy()
    got = got.reshape(qq.shape)
    kv = kk.shape[2]
    out_eps = 2.0 ** -23 if out.dtype == torch.float32 else EPS[ty]
    for i, s in enumerate(slots):
        n = int(lens[s]) if s >= 0 else 0
        pages = table[s, :-(-n // page)] if n else []
        k = kk[pages].reshape(-1, kv, hd)[:n]
        v = vv[pages].reshape(-1, kv, hd)[:n]
        want = R.attention(qq[i], k, v, n, t, scale)
        for j in range(t):
            seen = n - t + j + 1
            if seen <= 0:
                assert (got[i, j] == 0).all()
                continue
            kr, vr = (np.repeat(x[:seen], heads // kv, 1) for x in (k, v))
            x = np.einsum("hd,nhd->hn", qq[i, j], kr) * scale
            mag = np.einsum("hd,nhd->hn", abs(qq[i, j]), abs(kr)).max(1) * scale
            p = np.exp(x - x.max(1, keepdims=True))
            l1 = p.sum(1)
            p /= l1[:, None]
            carry = np.einsum("hn,nhd->hd", p, abs(vr))
            delta = (hd + 3) * 2.0 ** -24 * mag
            tol = carry * (EPS[ty] / 2 + 4 * delta[:, None] + 2.0 ** -20)
            if ty == F16:
                tol += abs(vr).sum(0) * 2.0 ** -25
            tol = tol * 1.01 + (abs(want[j]) + tol) * out_eps / 2 + 2.0 ** -25
            off = abs(got[i, j] - want[j])
            assert (off <= tol).all(), (i, j, s, n, float((off - tol).max()))


def queries(rng, rows, heads, hd, ty, sharp=1.0):
    return torch.from_numpy((sharp * rng.standard_normal((rows, heads, hd))).astype(np.float32)).to(TYPES[ty]).cuda()


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("sizes,shared,t,heads,kv,hd,page,ty", [
    ([[1]], [0], 1, 2, 1, 64, 16, BF16),
    ([[1, 16, 17, 0, 33]], [0], 1, 8, 2, 64, 16, F16),
    ([[5, 1, 0, 40]], [3], 1, 8, 2, 128, 16, BF16),
    ([[7, 300, 64]], [9], 1, 6, 2, 64, 64, F16),
    ([[3, 9, 4], [], [130], [20, 21]], [2, 1, 0, 5], 1, 4, 4, 64, 32, BF16),
    ([[3, 9, 4, 2, 1], [8, 1]], [2, 5], 4, 8, 2, 64, 32, F16),
    ([[0, 4, 4, 6]], [2], 4, 7, 1, 128, 16, BF16),          # a sequence that ends with the shared pages
    ([[1, 2, 2]], [0], 3, 4, 2, 64, 16, BF16),              # fewer positions than queries
    ([[11] * 40], [20], 1, 16, 2, 64, 16, BF16),
    ([[70] * 9, [1] * 30], [17, 33], 2, 24, 2, 128, 128, F16),
], ids=lambda v: str(v).replace(" ", "")[:28])
def test_attention(layer, layout, sizes, shared, t, heads, kv, hd, page, ty):
    rng = np.random.default_rng(len(sizes) * 100 + t)
    c, slots, bounds, lens, table = build_batch(layer, rng, sizes, shared, t, heads, kv, hd, page, ty, layout, pad=2)
    q = queries(rng, len(slots) * t, heads, hd, ty)
    out = run_attention(layer, c, slots, bounds, shared, t, heads, q)
    check_attention(c, slots, lens, table, t, heads, q, out)
    alone = run_attention(layer, c, slots, bounds, shared, t, heads, q, groups=False, out_type=0)
    check_attention(c, slots, lens, table, t, heads, q, alone)
    again = run_attention(layer, c, slots, bounds, shared, t, heads, q, max_len=1)
    check_attention(c, slots, lens, table, t, heads, q, again)
    assert torch.equal(out, run_attention(layer, c, slots, bounds, shared, t, heads, q))


@pytest.mark.parametrize("n,pages,own,t,heads,kv,hd,page,ty", [
    (1, 0, 5000, 1, 8, 1, 64, 16, BF16), (33, 70, 129, 1, 32, 8, 64, 64, BF16), (40, 65, 37, 2, 16, 2, 128, 32, F16),
    (130, 33, 9, 1, 8, 2, 64, 128, F16), (16, 129, 300, 1, 32, 4, 128, 16, BF16)])
def test_attention_longer(layer, n, pages, own, t, heads, kv, hd, page, ty):
    rng = np.random.default_rng(n)
    sizes = [[int(rng.integers(t, own + 1)) for _ in range(n)]]
    c, slots, bounds, lens, table = build_batch(layer, rng, sizes, [pages], t, heads, kv, hd, page, ty)
    q = queries(rng, n * t, heads, hd, ty, sharp=2.0)
    out = run_attention(layer, c, slots, bounds, [pages], t, heads, q)
    check_attention(c, slots, lens, table, t, heads, q, out)


def test_attention_shared_is_a_promise_cut_to_what_is_seen(layer):
    """More shared pages told than a sequence has, or than its first query sees: no other result."""
    rng = np.random.default_rng(21)
    c, slots, bounds, lens, table = build_batch(layer, rng, [[1, 40, 20], [17, 3]], [3, 2], 2, 4, 2, 64, 16, BF16)
    q = queries(rng, 10, 4, 64, BF16)
    want = run_attention(layer, c, slots, bounds, [0, 0], 2, 4, q)
    check_attention(c, slots, lens, table, 2, 4, q, want)
    for told in ([3, 2], [3, 1], [0, 2], [-5, 2]):
        out = run_attention(layer, c, slots, bounds, told, 2, 4, q)
        check_attention(c, slots, lens, table, 2, 4, q, out)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("t", [1, 3])
def test_attention_takes_nothing_from_behind(layer, value, t):
    """Whatever lies behind a query (the rest of its last page, later queries' rows, free pages) stays out
    of its result."""
    rng = np.random.default_rng(22)
    for sizes, shared in (([[5, 9, 37]], [2]), ([[2, 64, 18]], [0])):
        c, slots, bounds, lens, table = build_batch(layer, rng, sizes, shared, t, 8, 2, 64, 16, BF16)
        q = queries(rng, 3 * t, 8, 64, BF16)
        clean = run_attention(layer, c, slots, bounds, shared, t, 8, q)
        used = np.zeros((c.k.shape[1], 16), bool)
        for s in slots:
            for pos in range(lens[s]):
                used[table[s, pos // 16], pos % 16] = True
        dirt = torch.from_numpy(~used).cuda()
        for x in (c.k, c.v):
            x[1][dirt] = value
        assert torch.equal(clean, run_attention(layer, c, slots, bounds, shared, t, 8, q))
        if t == 3:
            # the last position of each sequence: only its last query sees it
            for s in slots:
                for x in (c.k, c.v):
                    x[1, table[s, (lens[s] - 1) // 16], (lens[s] - 1) % 16] = value
            got = run_attention(layer, c, slots, bounds, shared, t, 8, q).view(3, t, 8, 64)
            was = clean.view(3, t, 8, 64)
            assert torch.isfinite(got[:, :t - 1]).all()
            off = (got[:, :t - 1].float() - was[:, :t - 1].float()).abs().max()
            assert off <= 2 * EPS[BF16] * was.float().abs().max()
            assert torch.isnan(got[:, t - 1]).all() or value == -float("inf")


def test_attention_of_many_groups_and_sequences(layer):
    """More sequences than the rows kernel's estimate looks at, more groups than a warp has lanes, pads and
    empty sequences inside the groups, a scale below 0."""
    rng = np.random.default_rng(31)
    for groups, each, t, heads, scale in ((40, 4, 1, 8, None), (3, 50, 2, 4, -0.07), (1, 140, 1, 8, -0.2),
                                           (350, 3, 1, 4, None)):
        sizes = [[int(v) for v in rng.integers(t, 60, each)] for _ in range(groups)]
        for g in sizes:
            g[1] = t                       # as short as can be
        shared = [int(v) for v in rng.integers(0, 12, groups)]
        c, slots, bounds, lens, table = build_batch(layer, rng, sizes, shared, t, heads, 2, 64, 16, BF16)
        for g in range(groups):            # a pad and an emptied sequence in each group
            slots[bounds[g]] = -1 if g % 2 else len(lens) + 5
            lens[slots[bounds[g] + 2]] = 0
        c.len.copy_(torch.from_numpy(lens))
        q = queries(rng, len(slots) * t, heads, 64, BF16)
        q.view(len(slots), t, heads, 64)[bounds[0]] = float("nan")        # (what a pad holds)
        out = run_attention(layer, c, slots, bounds, shared, t, heads, q, scale=scale)
        known = [s if s < len(lens) else -1 for s in slots]
        check_attention(c, known, lens, table, t, heads, q, out, scale=scale)


def test_attention_of_as_many_sequences_and_groups_as_a_call_takes(layer):
    rng = np.random.default_rng(35)
    sizes = [[1 + (i + j) % 9 for j in range(16)] for i in range(4096)]
    c, slots, bounds, lens, table = build_batch(layer, rng, sizes, [1] * 4096, 1, 2, 1, 64, 16, BF16, layers=1, at=0)
    q = queries(rng, 65536, 2, 64, BF16)
    out = run_attention(layer, c, slots, bounds, [1] * 4096, 1, 2, q, at=0)
    some = np.concatenate((np.arange(40), np.arange(30000, 65536, 777), np.arange(65500, 65536)))
    check_attention(c, [slots[i] for i in some], lens, table, 1, 2, q[some], out[some], at=0)


def test_attention_with_a_scale_of_0(layer):
    """The mean of V over the keys that are seen, whichever kernel reads them: a prefix that ends inside a
    step of the tensor cores', and own keys; the smallest scale too."""
    rng = np.random.default_rng(34)
    for scale in (0.0, -0.0, 1e-45):
        c, slots, bounds, lens, table = build_batch(layer, rng, [[7] * 12], [5], 1, 8, 2, 64, 16, BF16)
        q = queries(rng, 12, 8, 64, BF16)
        out = run_attention(layer, c, slots, bounds, [5], 1, 8, q, scale=scale)
        check_attention(c, slots, lens, table, 1, 8, q, out, scale=scale)


def test_attention_of_a_whole_prompt(layer):
    """As many queries as positions, causal: the rows of a prompt, and of one that goes on from shared pages."""
    rng = np.random.default_rng(32)
    for n_tok, sizes, shared in ((90, [[90, 130, 200]], [0]), (60, [[60, 75]], [5])):
        c, slots, bounds, lens, table = build_batch(layer, rng, sizes, shared, n_tok, 4, 2, 64, 32, F16)
        q = queries(rng, len(slots) * n_tok, 4, 64, F16)
        out = run_attention(layer, c, slots, bounds, shared, n_tok, 4, q)
        check_attention(c, slots, lens, table, n_tok, 4, q, out)


@pytest.mark.parametrize("n_tok,sizes,shared,heads,kv,hd,page,ty", [
    (300, [[300, 420]], [0], 8, 2, 128, 16, BF16),
    (257, [[257]], [0], 4, 4, 128, 64, F16),
    (200, [[200, 260], [333]], [5, 0], 6, 2, 128, 32, BF16),
    (513, [[600]], [0], 4, 1, 64, 128, BF16)])
def test_attention_of_longer_prompts(layer, n_tok, sizes, shared, heads, kv, hd, page, ty):
    """Hundreds of queries a sequence, whole prompts and ones that go on, in both types and head sizes."""
    rng = np.random.default_rng(n_tok)
    c, slots, bounds, lens, table = build_batch(layer, rng, sizes, shared, n_tok, heads, kv, hd, page, ty)
    q = queries(rng, len(slots) * n_tok, heads, hd, ty)
    out = run_attention(layer, c, slots, bounds, shared, n_tok, heads, q)
    check_attention(c, slots, lens, table, n_tok, heads, q, out)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("hd,ty,t", [(128, BF16, 3), (128, F16, 40), (64, F16, 5)])
def test_attention_takes_nothing_from_later_queries(layer, value, hd, ty, t):
    """inf and NaN in the last position of a sequence, which only its last query sees: the others' bits stay those
    that they have with another finite V there."""
    rng = np.random.default_rng(24)
    c, slots, bounds, lens, table = build_batch(layer, rng, [[t, t + 9, t + 64]], [2], t, 8, 2, hd, 16, ty)
    q = queries(rng, 3 * t, 8, hd, ty)
    clean = run_attention(layer, c, slots, bounds, [2], t, 8, q).view(3, t, 8, hd)
    check_attention(c, slots, lens, table, t, 8, q, clean)
    for s in slots:
        c.v[1, table[s, (lens[s] - 1) // 16], (lens[s] - 1) % 16] = value
    got = run_attention(layer, c, slots, bounds, [2], t, 8, q).view(3, t, 8, hd)
    off = (got[:, :t - 1].float() - clean[:, :t - 1].float()).abs().max()
    assert off <= 2 * EPS[ty] * clean.float().abs().max()
    assert not torch.isfinite(got[:, t - 1]).any()


def test_attention_of_sequences_outside_the_groups(layer):
    """Groups that leave out the first and the last sequences and some between them, and a slot that is listed twice."""
    rng = np.random.default_rng(36)
    for hd, ty in ((64, F16), (128, BF16)):
        c, slots, _, lens, table = build_batch(layer, rng, [[30, 4], [9, 8, 7, 6], [77, 1], [5, 40, 3]], [0, 6, 3, 4], 2, 16, 2, hd, 16, ty)
        slots = slots + [slots[3], slots[0]]
        q = queries(rng, len(slots) * 2, 16, hd, ty)
        # group bounds are one list: what lies between two groups is a group that shares nothing
        for bounds, told in (([2, 6, 8, 11], [6, 0, 4]), ([3, 6], [6]), ([8, 11], [4])):
            out = run_attention(layer, c, slots, bounds, told, 2, 16, q)
            check_attention(c, slots, lens, table, 2, 16, q, out)


def test_attention_goes_by_the_lengths_of_the_replay(layer):
    """One captured call, replayed as the sequences, their groups and their shared pages change."""
    rng = np.random.default_rng(33)
    c, slots, bounds, lens, table = build_batch(layer, rng, [[40] * 9], [14], 1, 16, 2, 128, 16, BF16, spare=20)
    q = queries(rng, 9, 16, 128, BF16)
    out = torch.empty_like(q)
    sl, gr, sh = c.ints(slots), c.ints(bounds), c.ints([14])
    b = AttentionStruct(slots=sl.data_ptr(), group=gr.data_ptr(), shared=sh.data_ptr(), n_seq=9, n_tok=1, n_head=16,
                        n_group=1, max_len=300, out_type=BF16, scale=128 ** -0.5)
    w = scratch(layer.attention_work(c.p, b))
    b.work, b.work_bytes = w.data_ptr(), w.numel()
    side = torch.cuda.Stream()
    layer.attention_dev(c.p, 1, b, q.data_ptr(), out.data_ptr(), side.cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        layer.attention_dev(c.p, 1, b, q.data_ptr(), out.data_ptr(), side.cuda_stream)
    for told, cut in ((14, [40] * 9), (3, [40, 1, 17, 0, 40, 33, 2, 9, 16]), (0, [0] * 9), (14, [16, 40, 40, 40, 0, 8, 8, 8, 1])):
        for s, own in zip(slots, cut):
            lens[s] = 14 * 16 + own if own else (14 * 16 if told == 14 else 0)
        c.len.copy_(torch.from_numpy(lens))
        sh.fill_(told)
        q.copy_(queries(rng, 9, 16, 128, BF16))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check_attention(c, slots, lens, table, 1, 16, q, out)


def test_calls_on_two_streams_at_once(layer):
    """Attention and adapters on two streams, each with scratch of its own, many times over: the results of the
    calls alone."""
    rng = np.random.default_rng(34)
    jobs = []
    for hd, n in ((64, 24), (128, 12)):
        c, slots, bounds, lens, table = build_batch(layer, rng, [[30] * n], [40], 1, 16, 2, hd, 16, BF16)
        q = queries(rng, n, 16, hd, BF16)
        want = run_attention(layer, c, slots, bounds, [40], 1, 16, q)
        out = torch.empty_like(q)
        keep = [c.ints(slots), c.ints(bounds), c.ints([40])]
        b = AttentionStruct(slots=keep[0].data_ptr(), group=keep[1].data_ptr(), shared=keep[2].data_ptr(), n_seq=n, n_tok=1,
                            n_head=16, n_group=1, max_len=700, out_type=BF16, scale=hd ** -0.5)
        w = scratch(layer.attention_work(c.p, b))
        b.work, b.work_bytes = w.data_ptr(), w.numel()
        jobs.append((torch.cuda.Stream(), c, b, q, out, want.view_as(out), w, keep))
    torch.cuda.synchronize()
    for _ in range(40):
        for st_, c, b, q, out, *_ in jobs:
            layer.attention_dev(c.p, 1, b, q.data_ptr(), out.data_ptr(), st_.cuda_stream)
    torch.cuda.synchronize()
    for _, _, _, _, out, want, *_ in jobs:
        assert torch.equal(out, want)


def test_offsets_past_32_bits(layer):
    """A cache whose second layer lies past 2^32 elements: append, fork and attention there."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    rng = np.random.default_rng(35)
    c, slots, bounds, lens, table = build_batch(layer, rng, [[9, 20, 33]], [3], 1, 4, 2, 64, 16, BF16, layers=1)
    far = (1 << 32) + 4096
    need = far + c.k.numel()
    big = [torch.empty(need, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for x, pool in zip(big, (c.k, c.v)):
        x[:pool.numel()] = float("nan")
        x[far:] = pool.flatten()
    c.p.k, c.p.v, c.p.n_layer, c.p.layer_stride = big[0].data_ptr(), big[1].data_ptr(), 2, far
    c.k, c.v = [torch.stack((x[:pool.numel()].view(pool.shape[1:]), x[far:].view(pool.shape[1:]))) for x, pool in zip(big, (c.k, c.v))]
    q = queries(rng, 3, 4, 64, BF16)
    out = run_attention(layer, c, slots, bounds, [3], 1, 4, q, at=1)
    check_attention(c, slots, lens, table, 1, 4, q, out, at=1)
    # append one row to layer 1, fork it, and see both through the pool
    xs = [dev(rng.standard_normal((1, h * 64)).astype(np.float32)) for h in (4, 2, 2)]
    cs, q_out, sl = dev(rope_table(256, 64)), torch.zeros(1, 4, 64, dtype=torch.bfloat16, device="cuda"), c.ints([slots[0]])
    layer.pages_append_dev(c.p, 1, sl.data_ptr(), 1, 1, 4, *[x.data_ptr() for x in xs], cs.data_ptr(), 256, q_out.data_ptr(), st())
    ref = torch.zeros(c.p.n_pages, dtype=torch.int32)
    for s in slots:
        for j in range(-(-int(lens[s]) // 16)):
            ref[table[s, j]] += 1
    c.ref.copy_(ref)
    empty = next(s for s in range(len(lens)) if s not in slots)
    c.fork([slots[0]], [empty])
    torch.cuda.synchronize()
    pos = int(lens[slots[0]]) - 1
    new = c.table[empty, pos // 16].item()
    assert new != table[slots[0], pos // 16] and c.refused() == 0
    layer1 = big[1][far:].view(c.v.shape[1:])
    for page in (table[slots[0], pos // 16], new):
        assert torch.equal(layer1[page, pos % 16].flatten(), xs[2][0].bfloat16())


def test_attention_refusals(layer):
    rng = np.random.default_rng(2)
    c, slots, bounds, lens, table = build_batch(layer, rng, [[5, 9]], [1], 1, 4, 2, 64, 16, BF16)
    q = queries(rng, 2, 4, 64, BF16)
    out = torch.zeros_like(q)
    sl, gr, sh = c.ints(slots), c.ints(bounds), c.ints([1])

    def batch(**changes):
        b = AttentionStruct(slots=sl.data_ptr(), group=gr.data_ptr(), shared=sh.data_ptr(), n_seq=2, n_tok=1,
                            n_head=4, n_group=1, max_len=25, out_type=BF16, scale=0.125)
        w = scratch(layer.attention_work(c.p, b))
        b.work, b.work_bytes = w.data_ptr(), w.numel()
        for k, v in changes.items():
            setattr(b, k, v)
        return b, w

    b, w = batch()
    layer.attention_dev(c.p, 0, b, q.data_ptr(), out.data_ptr(), st())
    for changes in (dict(slots=None), dict(group=None), dict(shared=None), dict(n_tok=0), dict(n_head=0), dict(n_head=3),
                    dict(out_type=F16), dict(n_group=3), dict(work=None), dict(work_bytes=100), dict(n_seq=65537),
                    dict(n_seq=8192, n_group=4097), dict(n_tok=1 << 23)):
        b, w = batch(**changes)
        with pytest.raises(GpuError):
            layer.attention_dev(c.p, 0, b, q.data_ptr(), out.data_ptr(), st())
    for changes in (dict(n_seq=65537), dict(n_seq=8192, n_group=4097), dict(n_tok=1 << 23)):
        assert layer.attention_work(c.p, batch(**changes)[0]) == 0
    b, w = batch()
    for args in ((2, q.data_ptr(), out.data_ptr()), (0, 0, out.data_ptr()), (0, q.data_ptr(), out.data_ptr() + 2)):
        with pytest.raises(GpuError):
            layer.attention_dev(c.p, args[0], b, args[1], args[2], st())
    b, w = batch(n_seq=0, n_group=0)
    layer.attention_dev(c.p, 0, b, 0, 0, st())
    torch.cuda.synchronize()


def test_attention_scratch_fits_smaller_batches(layer):
    rng = np.random.default_rng(2)
    c, *_ = build_batch(layer, rng, [[5, 9]], [1], 1, 4, 2, 64, 16, BF16)

    def need(n, groups, t=1, max_len=4096):
        return layer.attention_work(c.p, AttentionStruct(slots=64, group=64, shared=64, n_seq=n, n_tok=t, n_head=32,
                                                         n_group=groups, max_len=max_len, out_type=0, scale=1))
    for t in (1, 3, 9):
        sizes = [need(n, min(n, 2), t) for n in range(1, 300)]
        assert sizes == sorted(sizes) and need(300, 1, t) <= need(300, 2, t)


# ---- adapters --------------------------------------------------------------------------


def make_adapters(rng, slots, max_rank, k, ns, ty, ranks=None):
    ranks = [int(v) for v in rng.integers(1, max_rank + 1, size=slots)] if ranks is None else ranks
    scale = (0.25 + rng.random(slots)).astype(np.float32)
    mats = []
    for n in ns:
        a = torch.from_numpy(rng.standard_normal((slots, max_rank, k)).astype(np.float32) * k ** -0.5).to(TYPES[ty])
        b = torch.from_numpy(rng.standard_normal((slots, n, max_rank)).astype(np.float32)).to(TYPES[ty])
        for s, r in enumerate(ranks):          # what lies behind a rank is not used
            a[s, r:] = float("nan")
            b[s, :, r:] = float("inf")
        mats.append((a, b))
    return mats, ranks, scale


def run_adapters(g, mats, ranks, scale, q, d, which, bases, in_place=False, ty=BF16):
    m, k = q.shape
    dm = [(a.cuda(), b.cuda()) for a, b in mats]
    rk, sc, wh = dev(np.array(ranks, np.int32)), dev(scale), dev(np.array(which, np.int32))
    sets = g.adapter_sets([AdaptersStruct(a=a.data_ptr(), b=b.data_ptr(), rank=rk.data_ptr(), scale=sc.data_ptr(),
                                          k=k, n=b.shape[1], slots=a.shape[0], max_rank=a.shape[1], type=ty)
                           for a, b in dm])
    db = [dev(b) for b in bases]
    ys = [torch.cat((b, torch.full((1, b.shape[1]), 9.0, device="cuda"))) if in_place else
          torch.full((m + 1, b.shape[1]), 9.0, device="cuda") for b in db]
    w = torch.full((g.adapters_work(sets, m) + 16,), 255, dtype=torch.uint8, device="cuda")
    dq, dd = dev(q), dev(d)
    g.adapters_dev(sets, m, dq.data_ptr(), dd.data_ptr(), wh.data_ptr(),
                   None if in_place else g.pointers([b.data_ptr() for b in db]),
                   g.pointers([y.data_ptr() for y in ys]), w.data_ptr(), w.numel() - 16, st())
    torch.cuda.synchronize()
    assert (w[-16:] == 255).all()
    for y in ys:
        assert (y[m] == 9).all()
    return [y[:m].cpu().numpy() for y in ys]


def check_adapters(q, d, which, mats, ranks, scale, bases, ys):
    """fp32: a 32-block's sum of exact products (32 roundings), k / 32 of them and the pieces joined, t's two
    tf32 parts (2^-21), the ranks' sum, the scale, the base: counted on the sums of magnitudes."""
    x = abs(q.astype(np.float64)) * np.repeat(d.astype(np.float64), 32, 1)
    for (a, b), base, y in zip(mats, bases, ys):
        a, b = a.double().numpy(), b.double().numpy()
        want = R.adapters(q, d, which, base, a, b, ranks, scale)
        tol = np.zeros_like(want)
        for r, s in enumerate(which):
            if 0 <= s < len(ranks):
                n = ranks[s]
                mag = abs(b[s][:, :n]) @ (abs(a[s][:n]) @ x[r]) * float(scale[s])
                roundings = 32 + q.shape[1] / 32 + 40 + 2 * n + 3
                tol[r] = mag * (roundings * 2.0 ** -23 + 2.0 ** -21) + abs(want[r]) * 2.0 ** -23
            else:
                assert np.array_equal(y[r].view(np.uint32), base[r].view(np.uint32))
        assert (abs(y - want) <= tol).all(), float((abs(y - want) - tol).max())


@pytest.mark.parametrize("m,k,ns,slots,max_rank,ty", [
    (1, 32, [1], 1, 4, BF16), (1, 2048, [2048, 512, 512], 4, 16, BF16), (3, 96, [7, 130], 2, 8, F16),
    (16, 1024, [129], 16, 24, F16), (17, 512, [64, 1], 3, 64, BF16), (33, 2048, [300], 40, 32, BF16),
    (70, 256, [1000], 2, 128, F16), (40, 128, [33], 5, 104, BF16), (600, 160, [96], 3, 40, F16),
    (5, 14336, [48], 5, 16, BF16), (560, 992, [130, 7], 70, 16, BF16), (513, 64, [64], 1, 8, F16),
    (530, 320, [201, 66], 4, 64, BF16), (300, 192, [130, 64], 3, 64, F16), (257, 64, [36], 9, 48, F16), (520, 32, [40], 3, 4, F16), (515, 96, [68], 2, 128, BF16)])
def test_adapters(layer, m, k, ns, slots, max_rank, ty):
    rng = np.random.default_rng(m + k)
    mats, ranks, scale = make_adapters(rng, slots, max_rank, k, ns, ty)
    q = rng.integers(-127, 128, (m, k)).astype(np.int8)
    d = (0.001 + 0.02 * rng.random((m, k // 32))).astype(np.float32)
    bases = [rng.standard_normal((m, n)).astype(np.float32) for n in ns]
    mixed = rng.integers(-1, slots + 1, m).tolist()        # -1 and `slots`: no adapter
    for which in (mixed, sorted(mixed), [-1] * m, [slots - 1] * m):
        for in_place in (False, True):
            ys = run_adapters(layer, mats, ranks, scale, q, d, which, bases, in_place, ty)
            check_adapters(q, d, which, mats, ranks, scale, bases, ys)


@pytest.mark.parametrize("m,max_ranks,ty", [
    (5, (4, 24), F16), (16, (64, 4), BF16), (21, (128, 4, 8), BF16), (33, (4, 32, 16), F16), (17, (8, 16, 4), BF16),
    (40, (8, 128), F16), (30, (24, 128, 64), BF16), (520, (4, 64), BF16), (530, (128, 4), F16), (515, (8, 64, 16), F16),
    (540, (64, 40), BF16)], ids=str)
def test_adapters_of_sets_of_different_rank(layer, m, max_ranks, ty):
    """Each set has a max_rank of its own, its columns of B as wide as that: odd N, ranks up to the whole
    of it, B's arrays as long as they have to be."""
    rng = np.random.default_rng(m + sum(max_ranks))
    k, slots, ns = 160, 5, [33, 130, 7][:len(max_ranks)]
    made = [make_adapters(rng, slots, r, k, [n], ty, ranks=[r, 1, 0, r, min(r, 3)]) for r, n in zip(max_ranks, ns)]
    dm = [(mats[0][0].cuda(), mats[0][1].cuda(), dev(np.array(ranks, np.int32)), dev(scale)) for mats, ranks, scale in made]
    sets = layer.adapter_sets([AdaptersStruct(a=a.data_ptr(), b=b.data_ptr(), rank=rk.data_ptr(), scale=sc.data_ptr(), k=k,
                                              n=b.shape[1], slots=slots, max_rank=a.shape[1], type=ty) for a, b, rk, sc in dm])
    q = rng.integers(-127, 128, (m, k)).astype(np.int8)
    d = (0.001 + 0.02 * rng.random((m, k // 32))).astype(np.float32)
    bases = [rng.standard_normal((m, n)).astype(np.float32) for n in ns]
    dq, dd, db = dev(q), dev(d), [dev(b) for b in bases]
    w = scratch(layer.adapters_work(sets, m))
    mixed = rng.integers(-1, slots + 1, m).tolist()
    for which in (mixed, sorted(mixed)):
        wh, ys = dev(np.array(which, np.int32)), [torch.full_like(b, 9.0) for b in db]
        layer.adapters_dev(sets, m, dq.data_ptr(), dd.data_ptr(), wh.data_ptr(), layer.pointers([b.data_ptr() for b in db]),
                           layer.pointers([y.data_ptr() for y in ys]), w.data_ptr(), w.numel(), st())
        torch.cuda.synchronize()
        for (mats, ranks, scale), base, y in zip(made, bases, ys):
            check_adapters(q, d, which, mats, ranks, scale, [base], [y.cpu().numpy()])


@pytest.mark.parametrize("m,k,ns,slots,max_rank,ty", [
    (128, 4096, [72], 4, 128, BF16), (128, 4096, [40], 3, 128, F16), (16, 4096, [40, 33], 6, 64, F16), (4, 4096, [50], 3, 128, BF16),
    (3, 4096, [50], 3, 128, F16), (600, 256, [130], 3, 128, F16)])
def test_adapters_whose_pieces_are_added_up_first(layer, m, k, ns, slots, max_rank, ty):
    """Short batches with many pieces of K and ranks enough that a launch of its own adds them up (and one on
    either side of that)."""
    rng = np.random.default_rng(m + max_rank)
    mats, ranks, scale = make_adapters(rng, slots, max_rank, k, ns, ty, ranks=[max_rank - i for i in range(slots)])
    q = rng.integers(-127, 128, (m, k)).astype(np.int8)
    d = (0.001 + 0.02 * rng.random((m, k // 32))).astype(np.float32)
    bases = [rng.standard_normal((m, n)).astype(np.float32) for n in ns]
    mixed = rng.integers(-1, slots + 1, m).tolist()
    for which in (mixed, [slots - 1] * m):
        ys = run_adapters(layer, mats, ranks, scale, q, d, which, bases, False, ty)
        check_adapters(q, d, which, mats, ranks, scale, bases, ys)


def test_adapters_rows_keep_apart(layer):
    """inf and NaN in one request's adapter, activation or base reach no other request; rank 0 adds 0, a rank out
    of range is cut to the table's."""
    rng = np.random.default_rng(4)
    m, k, n = 20, 256, 72
    mats, _, scale = make_adapters(rng, 5, 16, k, [n], BF16, ranks=[16, 3, 16, 16, 16])
    q = rng.integers(-127, 128, (m, k)).astype(np.int8)
    d = np.full((m, k // 32), 0.01, np.float32)
    base = rng.standard_normal((m, n)).astype(np.float32)
    which = [i % 4 for i in range(m)]
    clean = run_adapters(layer, mats, [16, 3, 0, 999, -3], scale, q, d, which, [base])
    check_adapters(q, d, which, mats, [16, 3, 0, 16, 0], scale, [base], clean)
    mats[0][0][0] = float("nan")
    mats[0][1][0] = float("inf")
    d[5] = np.inf
    got = run_adapters(layer, mats, [16, 3, 0, 999, -3], scale, q, d, which, [base])
    rows = [r for r in range(m) if which[r] != 0 and r != 5]
    assert np.array_equal(clean[0][rows], got[0][rows])


def test_adapters_rows_keep_apart_in_long_batches(layer):
    """The same where four tiles of rows pass together, two adapters at a time."""
    rng = np.random.default_rng(5)
    m, k, n = 600, 160, 68
    for ty in (F16, BF16):
        mats, _, scale = make_adapters(rng, 5, 16, k, [n], ty, ranks=[16, 3, 16, 16, 16])
        q = rng.integers(-127, 128, (m, k)).astype(np.int8)
        d = np.full((m, k // 32), 0.01, np.float32)
        base = rng.standard_normal((m, n)).astype(np.float32)
        which = [i % 5 - (i > 400) for i in range(m)]
        clean = run_adapters(layer, mats, [16, 3, 0, 999, -3], scale, q, d, which, [base], ty=ty)
        check_adapters(q, d, which, mats, [16, 3, 0, 16, 0], scale, [base], clean)
        mats[0][0][0] = float("nan")
        mats[0][1][0] = float("inf")
        d[5] = np.inf
        got = run_adapters(layer, mats, [16, 3, 0, 999, -3], scale, q, d, which, [base], ty=ty)
        rows = [r for r in range(m) if which[r] != 0 and r != 5]
        assert np.array_equal(clean[0][rows], got[0][rows])


@pytest.mark.parametrize("ty", [BF16, F16])
@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e4, 1e18])
def test_adapters_of_any_size_of_activation(layer, ty, size):
    """t far below and above what 16 bits hold, within a row too."""
    rng = np.random.default_rng(6)
    m, k, n, r = 520, 64, 72, 16
    mats, ranks, scale = make_adapters(rng, 2, r, k, [n], ty, ranks=[r, r])
    for s in range(2):
        mats[0][0][s] *= torch.tensor([10.0 ** (-i / 4) for i in range(r)])[:, None]
    q = rng.integers(-127, 128, (m, k)).astype(np.int8)
    d = (size * (0.1 + rng.random((m, k // 32)))).astype(np.float32)
    base = np.zeros((m, n), np.float32)
    which = rng.integers(0, 2, m).tolist()
    check_adapters(q, d, which, mats, ranks, scale, [base],
                   run_adapters(layer, mats, ranks, scale, q, d, which, [base], ty=ty))


@pytest.mark.parametrize("ty", [BF16, F16])
@pytest.mark.parametrize("m", [20, 520])
def test_adapters_of_infinite_t(layer, m, ty):
    """A t that passes fp32 gives outputs of B's sign and infinite, not NaN; what a rank leaves out adds 0 to
    an infinite activation too; a t next to fp32's largest is finite."""
    rng = np.random.default_rng(7)
    k, n, r = 64, 36, 16
    a = torch.zeros(4, r, k)
    a[:, 0, :32] = 1                       # t's first rank: the first block; the others: the second
    a[:, 1:, 32:] = torch.from_numpy(rng.standard_normal((4, r - 1, 32)).astype(np.float32))
    a[3, 0, 1:32] = 0                      # (adapter 3: one element of it)
    b = torch.from_numpy((np.sign(rng.standard_normal((4, n, r))) * (0.5 + rng.random((4, n, r)))).astype(np.float32))
    b[3] *= 2.0 ** -10
    mats, ranks, scale = [(a.to(TYPES[ty]), b.to(TYPES[ty]))], [16, 16, 0, 16], np.ones(4, np.float32)
    q = rng.integers(1, 128, (m, k)).astype(np.int8)
    q[:, 0] = 127
    d = (0.01 + 0.01 * rng.random((m, k // 32))).astype(np.float32)
    which = [i % 5 - 1 for i in range(m)]
    kind = [(i // 5) % 4 for i in range(m)]
    for i in range(m):
        if which[i] == 3:                  # finite, but more than the largest bf16 and its half step
            d[i, 0] = [3.4e38 / 127, 3.395e38 / 127, 3.397e38 / 127, 1][kind[i]]
        else:
            d[i, 0] = [np.inf, 3e37, -np.inf, 0.01][kind[i]]
    base = rng.standard_normal((m, n)).astype(np.float32)
    y = run_adapters(layer, mats, ranks, scale, q, d, which, [base], ty=ty)[0]
    sign = np.sign(b.numpy()[:, :, 0])
    plain = [i for i in range(m) if which[i] in (0, 1) and kind[i] == 3 or which[i] in (-1, 3)]
    check_adapters(q[plain], d[plain], [which[i] for i in plain], mats, ranks, scale, [base[plain]], [y[plain]])
    for i in range(m):
        if which[i] == 2:
            assert np.array_equal(y[i], base[i])
        elif which[i] in (0, 1) and kind[i] == 1:
            assert np.array_equal(y[i], sign[which[i]] * np.float32(np.inf)), i
        elif which[i] in (0, 1) and kind[i] != 3:
            assert np.isnan(y[i]).all(), i     # (inf times A's zeros in the other ranks)


@pytest.mark.parametrize("ty", [BF16, F16])
@pytest.mark.parametrize("m", [20, 520])
def test_adapters_of_infinite_activations(layer, m, ty):
    """An infinite d: every t is infinite, so y is where B's row has one sign, and NaN where it has both."""
    rng = np.random.default_rng(8)
    k, n, r = 96, 40, 24
    a = torch.from_numpy((0.1 + rng.random((2, r, k))).astype(np.float32))
    sign = rng.choice([-1, 1], (2, n)).astype(np.float32)
    b = (0.1 + rng.random((2, n, r))).astype(np.float32) * sign[:, :, None]
    b[:, ::7, 5] *= -1
    mats, ranks, scale = [(a.to(TYPES[ty]), torch.from_numpy(b).to(TYPES[ty]))], [24, 19], np.ones(2, np.float32)
    q = rng.integers(1, 128, (m, k)).astype(np.int8)
    d = (0.01 + 0.01 * rng.random((m, k // 32))).astype(np.float32)
    hot = rng.random(m) < 0.5
    d[hot, 1] = np.where(rng.random(m) < 0.5, np.inf, -np.inf)[hot]
    which = (np.arange(m) % 3 - 1).tolist()
    base = rng.standard_normal((m, n)).astype(np.float32)
    y = run_adapters(layer, mats, ranks, scale, q, d, which, [base], ty=ty)[0]
    cold = [i for i in range(m) if not hot[i] or which[i] < 0]
    check_adapters(q[cold], d[cold], [which[i] for i in cold], mats, ranks, scale, [base[cold]], [y[cold]])
    for i in range(m):
        if hot[i] and which[i] >= 0:
            want = sign[which[i]] * d[i, 1]
            want[::7] = np.nan
            assert np.array_equal(y[i], want, equal_nan=True), i


def test_adapters_refusals(layer):
    rng = np.random.default_rng(6)
    mats, ranks, scale = make_adapters(rng, 2, 8, 64, [10], BF16)
    a, b = mats[0][0].cuda(), mats[0][1].cuda()
    rk, sc = dev(np.array(ranks, np.int32)), dev(scale)
    q, d, y = torch.zeros(2, 64, dtype=torch.int8, device="cuda"), torch.zeros(2, 2, device="cuda"), torch.zeros(2, 10, device="cuda")
    wh = dev(np.array([0, 1], np.int32))
    w = scratch(1 << 20)

    def sets(count=1, **changes):
        s = AdaptersStruct(a=a.data_ptr(), b=b.data_ptr(), rank=rk.data_ptr(), scale=sc.data_ptr(), k=64, n=10, slots=2,
                           max_rank=8, type=BF16)
        for key, v in changes.items():
            setattr(s, key, v)
        return layer.adapter_sets([s] * count)

    def call(s, **changes):
        args = dict(m=2, q=q.data_ptr(), d=d.data_ptr(), which=wh.data_ptr(), bases=None,
                    ys=layer.pointers([y.data_ptr()] * len(s)), work=w.data_ptr(), work_bytes=w.numel(), stream=st())
        args.update(changes)
        layer.adapters_dev(s, **args)

    call(sets())
    call(sets(), m=0)
    for changes in (dict(a=None), dict(b=None), dict(rank=None), dict(scale=None), dict(k=48), dict(k=0), dict(n=0),
                    dict(max_rank=0), dict(max_rank=12), dict(max_rank=136), dict(type=0), dict(a=a.data_ptr() + 2)):
        assert layer.adapters_work(sets(**changes), 2) == 0
        with pytest.raises(GpuError):
            call(sets(**changes))
    with pytest.raises(GpuError):
        call(sets(count=9))
    other = torch.zeros(2, 10, device="cuda")
    two = layer.pointers([y.data_ptr(), other.data_ptr()])
    call(sets(count=2), ys=two)
    call(sets(count=2), ys=two, bases=two)
    with pytest.raises(GpuError):                        # one output of two sets
        call(sets(count=2), ys=layer.pointers([y.data_ptr()] * 2))
    with pytest.raises(GpuError):                        # a base that is the other's output
        call(sets(count=2), ys=two, bases=layer.pointers([other.data_ptr(), y.data_ptr()]))
    for changes in (dict(q=0), dict(q=q.data_ptr() + 8), dict(d=0), dict(which=0), dict(work=0), dict(work_bytes=64),
                    dict(ys=layer.pointers([0])), dict(work=w.data_ptr() + 4), dict(m=(1 << 24) + 1)):
        with pytest.raises(GpuError):
            call(sets(), **changes)
    sizes = [layer.adapters_work(sets(), m) for m in range(1, 6000, 7)]
    assert sizes == sorted(sizes)
    torch.cuda.synchronize()


def test_adapters_scratch_of_refused_sizes_is_0(layer):
    """The size of the scratch says what the call would: more rows or columns than it takes are 0 there too."""
    rng = np.random.default_rng(6)
    mats, ranks, scale = make_adapters(rng, 2, 8, 64, [10], BF16)
    a, b = mats[0][0].cuda(), mats[0][1].cuda()
    rk, sc, some = dev(np.array(ranks, np.int32)), dev(scale), torch.zeros(64, device="cuda")

    def sets(n, max_rank=8):
        return layer.adapter_sets([AdaptersStruct(a=a.data_ptr(), b=b.data_ptr(), rank=rk.data_ptr(), scale=sc.data_ptr(),
                                                  k=64, n=n, slots=2, max_rank=max_rank, type=BF16)])
    assert layer.adapters_work(sets(10), 1 << 24) > 0 and layer.adapters_work(sets(10), (1 << 24) + 1) == 0
    wide = 256 * 65535
    for n, m in ((wide, 16), (wide, 400), (4 * wide, 600)):      # (600 rows: 64 a CTA, up to 1024 columns)
        assert layer.adapters_work(sets(n), m) > 0
        assert layer.adapters_work(sets(n + 1), m) == 0
        with pytest.raises(GpuError):
            layer.adapters_dev(sets(n + 1), m, some.data_ptr(), some.data_ptr(), some.data_ptr(), None,
                               layer.pointers([some.data_ptr()]), some.data_ptr(), 1 << 62, st())


# ---- all together --------------------------------------------------------------------------


def test_a_batched_step(layer):
    """Three steps of six sequences (two groups forked from two prompts) through one layer's attention block: norm,
    the projections with adapters, append, attention, the output projection -- eagerly, and the same steps as
    replays of one captured graph. The graph's bits are the eager ones; every operator's result is held to its own
    plain form on the inputs that it got."""
    n_embd, heads, kv, hd, n = 256, 4, 2, 64, 6
    rng = np.random.default_rng(77)
    wq = {}
    for name, (k, rows) in dict(q=(n_embd, heads * hd), k=(n_embd, kv * hd), v=(n_embd, kv * hd), o=(heads * hd, n_embd)).items():
        blk, _ = W.matvec_inputs(G.GGML_Q8_0, k, rows, seed=len(wq))
        wq[name] = layer.add_blocks(G.GGML_Q8_0, k, rows, blk, "step." + name)
    mats, ranks, scale = make_adapters(rng, 3, 8, n_embd, [heads * hd, kv * hd, kv * hd], BF16)
    gain = dev((1 + 0.1 * rng.standard_normal(n_embd)).astype(np.float32))
    cs = rope_table(256, hd)
    dcs = dev(cs)

    def fresh():
        g = np.random.default_rng(5)
        c = Cache(layer, g, n_seq=8, max_pages=8, n_pages=40, kv=kv, hd=hd, layers=1)
        c.grow([0, 1], 70)
        c.fork([0, 0, 0, 1, 1], [2, 3, 4, 5, 6])
        c.free([0])
        torch.cuda.synchronize()
        return c

    def buffers():
        f = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
        return dict(x=f(n, n_embd), add=f(n, n_embd), q8=torch.zeros(n, n_embd, dtype=torch.int8, device="cuda"),
                    d8=f(n, n_embd // 32), yq=f(n, heads * hd), yk=f(n, kv * hd), yv=f(n, kv * hd),
                    qr=torch.zeros(n, heads, hd, dtype=torch.bfloat16, device="cuda"), at=f(n, heads * hd),
                    a8=torch.zeros(n, heads * hd, dtype=torch.int8, device="cuda"), ad=f(n, heads * hd // 32), yo=f(n, n_embd))

    dm = [(a.cuda(), b.cuda()) for a, b in mats]
    rk, sc = dev(np.array(ranks, np.int32)), dev(scale)
    which = [0, 2, -1, 1, 1, 0]
    wh = dev(np.array(which, np.int32))
    slots = [2, 3, 4, 1, 5, 6]
    sl, gr, sh = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (slots, [0, 3, 6], [4, 4]))

    def step(c, b, stream):
        sets = layer.adapter_sets([AdaptersStruct(a=a.data_ptr(), b=bb.data_ptr(), rank=rk.data_ptr(), scale=sc.data_ptr(),
                                                  k=n_embd, n=bb.shape[1], slots=3, max_rank=8, type=BF16) for a, bb in dm])
        ys = [b["yq"].data_ptr(), b["yk"].data_ptr(), b["yv"].data_ptr()]
        batch = AttentionStruct(slots=sl.data_ptr(), group=gr.data_ptr(), shared=sh.data_ptr(), n_seq=n, n_tok=1, n_head=heads,
                                n_group=2, max_len=128, out_type=0, scale=hd ** -0.5)
        if "w" not in b:
            b["w"] = scratch(layer.attention_work(c.p, batch))
            b["wa"] = scratch(layer.adapters_work(sets, n))
        batch.work, batch.work_bytes = b["w"].data_ptr(), b["w"].numel()
        layer.pages_grow_dev(c.p, sl.data_ptr(), n, 1, stream)
        layer.norm_quantise_dev(b["x"].data_ptr(), b["add"].data_ptr(), gain.data_ptr(), n, n_embd, 1e-5, b["x"].data_ptr(),
                                b["q8"].data_ptr(), b["d8"].data_ptr(), stream)
        assert layer.batch_group_dev([wq["q"], wq["k"], wq["v"]], n, b["q8"].data_ptr(), b["d8"].data_ptr(), ys, stream) == 0
        layer.adapters_dev(sets, n, b["q8"].data_ptr(), b["d8"].data_ptr(), wh.data_ptr(), None, layer.pointers(ys),
                           b["wa"].data_ptr(), b["wa"].numel(), stream)
        layer.pages_append_dev(c.p, 0, sl.data_ptr(), n, 1, heads, *ys, dcs.data_ptr(), 256, b["qr"].data_ptr(), stream)
        layer.attention_dev(c.p, 0, batch, b["qr"].data_ptr(), b["at"].data_ptr(), stream)
        assert layer.act_quantise_dev(b["at"].data_ptr(), n, heads * hd, b["a8"].data_ptr(), b["ad"].data_ptr(), stream) == 0
        assert layer.batch_group_dev([wq["o"]], n, b["a8"].data_ptr(), b["ad"].data_ptr(), [b["yo"].data_ptr()], stream) == 0

    xs = [dev(rng.standard_normal((n, n_embd)).astype(np.float32)) for _ in range(3)]
    side = torch.cuda.Stream()
    c, b = fresh(), buffers()
    eager = []
    for x in xs:
        with torch.cuda.stream(side):
            b["x"].copy_(x)
            b["add"].copy_(b["yo"])
            add = b["yo"].cpu().numpy().copy()
            lens0 = c.len.cpu().numpy().copy()
            step(c, b, side.cuda_stream)
        torch.cuda.synchronize()
        eager.append({k: v.clone() for k, v in b.items() if k not in ("w", "wa")})
        # each operator on what it got
        s, q8, d8 = R.norm_rows(x.cpu().numpy(), add, gain.cpu().numpy(), 1e-5)
        assert np.array_equal(b["q8"].cpu().numpy(), q8) and np.array_equal(b["d8"].cpu().numpy(), d8)
        assert np.array_equal(b["x"].cpu().numpy(), s)
        lens, table = c.len.cpu().numpy(), c.table.cpu().numpy()
        assert [lens[i] - lens0[i] for i in range(8)] == [1 if i in slots else 0 for i in range(8)]
        for i, slot in enumerate(slots):
            pos = int(lens[slot]) - 1
            key = torch.from_numpy(turn32(b["yk"][i].cpu().numpy().reshape(kv, hd), cs[pos])).to(torch.bfloat16)
            assert torch.equal(c.k[0, table[slot, pos // 16], pos % 16].cpu(), key)
        check_attention(c, slots, lens, table, 1, heads, b["qr"], b["at"].view(n, heads, hd), at=0)
        oq, od = O.act_quantise(b["at"][0].cpu().numpy())
        assert np.array_equal(b["a8"][0].cpu().numpy(), oq)
    assert c.refused() == 0

    c2, b2 = fresh(), buffers()
    with torch.cuda.stream(side):
        step(c2, b2, side.cuda_stream)          # once before capture: first-use set-up
        torch.cuda.synchronize()
    keep = b2["w"], b2["wa"]
    c2 = fresh()
    for k, v in buffers().items():
        b2[k].copy_(v)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        step(c2, b2, side.cuda_stream)
    for x, want in zip(xs, eager):
        b2["x"].copy_(x)
        b2["add"].copy_(b2["yo"])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for k, v in want.items():
            assert torch.equal(v, b2[k]), k
    assert torch.equal(c.len, c2.len) and torch.equal(c.ref, c2.ref) and torch.equal(c.k, c2.k) and torch.equal(c.v, c2.v)
    del keep
