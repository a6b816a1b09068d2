"""The paged cache on a GPU against plain implementations in 64 bits: append, attention, observed weights, eviction, and a run of them together.

Bounds.  A score of D products, summed in 32 bits in any order, is off by at most (D + 4) 2^-23 sum |q_d k_d| (every addition rounded or cut
off), a weight by twice that and 2^-20 relatively (the exponential and its argument), the sum over n positions by n 2^-23.  From a bf16 pool every
weight is rounded by 2^-8 (half a step) before it meets the values; results of 16 bits are rounded by 2^-8 once more."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class _Memory:
    def __init__(self, pool, ptr, shape, typestr):
        self.pool = pool  # lives as long as what looks at its memory
        self.__cuda_array_interface__ = dict(data=(ptr, False), shape=shape, typestr=typestr, version=3)


class World:
    """A pool full of what earlier sequences may have left (NaN and infinities), and sequences with their pages."""

    def __init__(self, L, dtype, heads, page, q_lens, kv_lens, seed=0, spare=3, extra=None):
        self.L, self.dtype, self.page = L, dtype, page
        self.Hq, self.Hkv, self.D = heads
        self.t = torch.bfloat16 if dtype == "bf16" else torch.float32
        self.g = torch.Generator(device=DEV).manual_seed(seed)
        self.q_lens, self.kv_lens = list(q_lens), list(kv_lens)
        need = [-(-k // page) for k in kv_lens] + [-(-k // page) for k in extra or []]
        self.pages = max(1, sum(need) + spare)
        order = np.random.default_rng(seed).permutation(self.pages)
        ends = np.cumsum(need)
        tables = [order[e - n: e].tolist() for e, n in zip(ends, need)]
        self.tables, self.extra_tables = tables[: len(kv_lens)], tables[len(kv_lens):]
        self.pool = L.PagePool(self.pages, page, self.Hkv, self.D, L.BF16 if dtype == "bf16" else L.F32)
        self.pool.ctx.synchronize()
        look = lambda ptr, shape, ty: torch.as_tensor(_Memory(self.pool, ptr, shape, ty), device=DEV)  # noqa: E731
        self.k, self.v = (look(p, self.pool.shape, "<i2" if dtype == "bf16" else "<f4").view(self.t) for p in (self.pool.k_ptr, self.pool.v_ptr))
        self.mass = look(self.pool.mass_ptr, self.pool.shape[:3], "<f4")
        assert not self.k.any() and not self.v.any() and not self.mass.any()
        self.k.fill_(float("nan"))
        self.v.fill_(float("inf"))
        self.v[:, :, ::2] = float("nan")
        self.mass.fill_(float("nan"))
        for b, n in enumerate(kv_lens):
            self.put(self.k, b, self.randn(n, self.Hkv, self.D))
            self.put(self.v, b, self.randn(n, self.Hkv, self.D))
            self.put(self.mass, b, torch.rand(n, self.Hkv, generator=self.g, device=DEV))

    def randn(self, *shape):
        return torch.randn(shape, generator=self.g, device=DEV)

    def at(self, table, n):
        pos = np.arange(n)
        return torch.as_tensor(np.asarray(table, np.int64)[pos // self.page] if n else pos, device=DEV), torch.as_tensor(pos % self.page, device=DEV)

    def put(self, pool, b, rows):
        page, slot = self.at(self.tables[b], rows.shape[0])
        pool[page, :, slot] = rows.to(pool.dtype)

    def rows(self, pool, table, n):
        page, slot = self.at(table, n)
        return pool[page, :, slot]

    def batch(self, q_lens=None, kv_lens=None, tables=None, **kw):
        return self.L.PageBatch(self.pool, self.Hq, self.q_lens if q_lens is None else q_lens, self.kv_lens if kv_lens is None else kv_lens,
                                self.tables if tables is None else tables, **kw)


def reference(w, q, scale, causal=True, q_lens=None, kv_lens=None, tables=None, out_bits=True):
    """Outputs, log-sums, weights received per sequence and the bounds of the first two, in 64 bits."""
    q_lens, kv_lens, tables = q_lens or w.q_lens, kv_lens or w.kv_lens, tables or w.tables
    G, t = w.Hq // w.Hkv, 0
    outs, lses, tols, ltols, mass = [], [], [], [], []
    for b, n in enumerate(q_lens):
        k, v = (w.rows(x, tables[b], kv_lens[b]).double() for x in (w.k, w.v))
        x = q[t: t + n].double()
        t += n
        kk, vv = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)  # [kv, Hq, D]
        s = torch.einsum("thd,jhd->htj", x, kk) * scale
        big = torch.einsum("thd,jhd->htj", x.abs(), kk.abs()) * abs(scale)
        seen = torch.ones(n, kv_lens[b], dtype=torch.bool, device=DEV)
        if causal:
            seen = torch.arange(kv_lens[b], device=DEV)[None] <= kv_lens[b] - n + torch.arange(n, device=DEV)[:, None]
        s = s.masked_fill(~seen, -np.inf)
        if kv_lens[b] == 0:
            outs.append(torch.zeros(n, w.Hq, w.D, dtype=torch.float64))
            lses.append(torch.full((n, w.Hq), -np.inf, dtype=torch.float64))
            tols.append(torch.zeros_like(outs[-1]))
            ltols.append(torch.zeros(n, w.Hq, dtype=torch.float64))
            mass.append(None)
            continue
        p = torch.softmax(s, -1)
        ds = (w.D + 4) * 2.0 ** -23 * (big * seen).amax(-1, keepdim=True)  # of a score of the row
        rel = 2 * ds + 2.0 ** -20 + kv_lens[b] * 2.0 ** -23
        av = torch.einsum("htj,jhd->thd", p, vv.abs())
        rel_t = rel.squeeze(-1).T[:, :, None]
        o = torch.einsum("htj,jhd->thd", p, vv)
        tol = av * (2 * rel_t + (2.0 ** -8 if w.dtype == "bf16" else 0)) + (o.abs() * 2.0 ** -8 if w.dtype == "bf16" and out_bits else 0) + 1e-30
        outs.append(o.cpu())
        tols.append(tol.cpu())
        lse = torch.logsumexp(s, -1)
        lses.append(lse.T.cpu())
        ltols.append((rel.squeeze(-1) + lse.abs() * 2.0 ** -21).T.cpu())
        mass.append((p.view(w.Hkv, G, n, kv_lens[b]).sum((1, 2)).T.cpu(), (p * 2 * (rel + ds)).view(w.Hkv, G, n, kv_lens[b]).sum((1, 2)).T.cpu() + n * G * 1e-7))
    return torch.cat(outs), torch.cat(lses), torch.cat(tols), torch.cat(ltols), mass


def attend(w, q, scale, causal=True, out=None, **kw):
    batch = w.batch(causal=causal, **kw)
    out = torch.full((q.shape[0] + 2, w.Hq, w.D), 77.0, dtype=out or w.t, device=DEV)
    lse = torch.full((q.shape[0] + 2, w.Hq), 77.0, device=DEV)
    torch.cuda.synchronize()
    w.L.paged_attention(w.pool, batch, q.data_ptr(), scale, out.data_ptr(), out_dtype=w.L.F32 if out.dtype == torch.float32 else w.L.BF16, lse_ptr=lse.data_ptr())
    w.pool.ctx.synchronize()
    assert (out[-2:] == 77).all() and (lse[-2:] == 77).all()  # what lies behind the last token stays
    return out[:-2].double().cpu(), lse[:-2].double().cpu(), batch


def close(got, want, tol):
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    d = (got - want)[~inf].abs()
    assert not d.isnan().any() and (d <= tol[~inf]).all(), float((d / tol[~inf]).max())


HEADS = [(8, 2, 64), (7, 1, 128), (4, 4, 64), (32, 8, 128), (40, 1, 64)]
LENS = [
    ([1], [1]), ([1, 1, 1, 1, 1, 1], [1, 63, 64, 65, 128, 2047]), ([0, 5, 0, 1, 0], [9, 5, 0, 130, 0]), ([17, 1, 128, 33], [17, 300, 129, 1000]),
    ([257, 64, 2], [257, 700, 2]),
]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("lens", range(len(LENS)))
def test_attention(L, dtype, heads, lens):
    q_lens, kv_lens = LENS[lens]
    w = World(L, dtype, heads, [8, 16, 32, 64, 128, 256][(lens + heads[0]) % 6], q_lens, kv_lens, seed=lens)
    q = w.randn(sum(q_lens), w.Hq, w.D).mul_(2).to(w.t)
    out, lse, _ = attend(w, q, w.D ** -0.5)
    o, l, to, tl, _ = reference(w, q, w.D ** -0.5)
    close(out, o, to)
    close(lse, l, tl)


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_pages_of_all_sizes(L, dtype, page):
    q_lens, kv_lens = [1, 70, 3], [page - 1, 4 * page + 71, 2 * page]
    w = World(L, dtype, (8, 2, 128), page, q_lens, kv_lens, seed=page)
    q = w.randn(sum(q_lens), w.Hq, w.D).to(w.t)
    out, lse, _ = attend(w, q, 0.11)
    o, l, to, tl, _ = reference(w, q, 0.11)
    close(out, o, to)
    close(lse, l, tl)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads", [(32, 8, 128), (4, 4, 64), (8, 1, 64)], ids=str)
@pytest.mark.parametrize("q_len", [1, 3, 40, 300])
def test_long_contexts_are_cut_and_joined(L, dtype, heads, q_len):
    w = World(L, dtype, heads, 64, [q_len, 1], [5003, 900], seed=q_len)
    q = w.randn(q_len + 1, w.Hq, w.D).mul_(2).to(w.t)
    out, lse, _ = attend(w, q, w.D ** -0.5)
    o, l, to, tl, _ = reference(w, q, w.D ** -0.5)
    close(out, o, to)
    close(lse, l, tl)


@pytest.mark.parametrize("dtype,heads,q_len,kv_len", [("bf16", (8, 8, 64), 5000, 5000), ("bf16", (32, 8, 128), 1400, 3100), ("f32", (8, 8, 64), 2500, 2700)])
def test_more_items_than_run_at_once(L, dtype, heads, q_len, kv_len):
    """The items of the last round are cut, and joined."""
    w = World(L, dtype, heads, 64, [q_len, 1], [kv_len, 70])
    q = w.randn(q_len + 1, w.Hq, w.D).mul_(2).to(w.t)
    out, lse, _ = attend(w, q, w.D ** -0.5)
    o, l, to, tl, _ = reference(w, q, w.D ** -0.5)
    close(out, o, to)
    close(lse, l, tl)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("singles", [3, 24])
def test_single_tokens_beside_a_chunk(L, dtype, singles):
    """With the chunk's rows, or, where there is more to read, in a launch of their own."""
    q_lens, kv_lens = [1] * singles + [100] + [2], [390 + i for i in range(singles)] + [500, 410]
    w = World(L, dtype, (32, 8, 128), 64, q_lens, kv_lens)
    q = w.randn(sum(q_lens), w.Hq, w.D).to(w.t)
    out, lse, _ = attend(w, q, w.D ** -0.5)
    o, l, to, tl, _ = reference(w, q, w.D ** -0.5)
    close(out, o, to)
    close(lse, l, tl)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("q_len,kv_len", [(1, 500), (20, 500), (200, 700)])
@pytest.mark.parametrize("at", [3, 64, 130, 499])
def test_a_key_that_is_no_number(L, dtype, q_len, kv_len, at):
    """Tokens that see it have no finite result, the others what they had."""
    w = World(L, dtype, (8, 2, 64), 16, [q_len], [kv_len])
    q = w.randn(q_len, w.Hq, w.D).to(w.t)
    before, _, _ = attend(w, q, 0.125)
    page, slot = w.at(w.tables[0], kv_len)
    w.k[page[at], :, slot[at]] = float("nan")
    after, lse, _ = attend(w, q, 0.125)
    sees = torch.arange(q_len) + kv_len - q_len >= at
    assert torch.equal(after[~sees], before[~sees])
    assert not torch.isfinite(after[sees]).any() and not torch.isfinite(lse[sees]).any()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_pool_beyond_32_bits(L, dtype):
    """More than 2^32 bytes and 2^31 numbers of keys; the sequences' pages lie all over it."""
    heads, page = (8, 4, 128), 64
    q_lens, kv_lens = [1, 90, 2], [700, 300, 64]
    w = World(L, dtype, heads, page, q_lens, kv_lens, spare=3 * 2 ** 30 // (4 * 128 * 64), extra=[100, 64, 1])
    assert max(map(max, w.tables)) * 4 * 128 * 64 > 2 ** 31
    q = w.randn(sum(q_lens), w.Hq, w.D).to(w.t)
    qkv = w.randn(sum(q_lens), 16 * 128)
    batch = w.batch()
    q_out = torch.empty(sum(q_lens), 8, 128, dtype=w.t, device=DEV)
    torch.cuda.synchronize()
    at = qkv.data_ptr()
    L.paged_append(w.pool, batch, at, at + 4 * 8 * 128, at + 4 * 12 * 128, 16 * 128, 16 * 128, q_out.data_ptr())
    w.pool.ctx.synchronize()
    t = 0
    for b, n in enumerate(q_lens):
        assert torch.equal(w.rows(w.k, w.tables[b], kv_lens[b])[kv_lens[b] - n:], qkv[t: t + n, 8 * 128: 12 * 128].view(n, 4, 128).to(w.t))
        t += n
    before = [w.rows(w.mass, w.tables[b], n).double().cpu() for b, n in enumerate(kv_lens)]
    out, lse, _ = attend(w, q, w.D ** -0.5)
    o, l, to, tl, mass = reference(w, q, w.D ** -0.5)
    close(out, o, to)
    close(lse, l, tl)
    dev_lse = lse.float().to(DEV)
    torch.cuda.synchronize()
    L.paged_attention_mass(w.pool, batch, q.data_ptr(), w.D ** -0.5, dev_lse.data_ptr())
    w.pool.ctx.synchronize()
    for b, n in enumerate(kv_lens):
        close(w.rows(w.mass, w.tables[b], n).double().cpu(), before[b] + mass[b][0], mass[b][1] + (before[b] + mass[b][0]) * 2.0 ** -22)
    kept = torch.zeros(3, 4, 100, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    L.paged_evict(w.pool, batch, w.batch(q_lens=[0] * 3, kv_lens=[100, 64, 1], tables=w.extra_tables), 5, kept.data_ptr(), 100)
    w.pool.ctx.synchronize()
    for b, n in enumerate([100, 64, 1]):
        for pool in (w.k, w.v):
            was, now = w.rows(pool, w.tables[b], kv_lens[b]), w.rows(pool, w.extra_tables[b], n)
            for h in range(4):
                assert torch.equal(now[:, h], was[kept[b, h, :n].long(), h])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_without_a_causal_mask(L, dtype):
    """Every token sees all positions; more tokens than positions, and none at all (zeros and -infinity)."""
    q_lens, kv_lens = [5, 3, 200, 1], [70, 0, 130, 0]
    w = World(L, dtype, (8, 2, 64), 16, q_lens, kv_lens)
    q = w.randn(sum(q_lens), w.Hq, w.D).to(w.t)
    out, lse, _ = attend(w, q, 0.3, causal=False)
    o, l, to, tl, _ = reference(w, q, 0.3, causal=False)
    close(out, o, to)
    close(lse, l, tl)
    assert not out[5:8].any()


@pytest.mark.parametrize("q_len,kv_len", [(1, 100), (130, 700)])
def test_f32_results_from_a_bf16_pool(L, q_len, kv_len):
    w = World(L, "bf16", (8, 2, 128), 32, [q_len], [kv_len])
    q = w.randn(q_len, w.Hq, w.D).to(w.t)
    out, _, _ = attend(w, q, w.D ** -0.5, out=torch.float32)
    o, _, to, _, _ = reference(w, q, w.D ** -0.5, out_bits=False)
    close(out, o, to)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [0.0, -0.2, 4.0])
def test_scales(L, dtype, scale):
    """0: the mean of what is seen; large ones: rows that a few positions fill, running maxima that grow by hundreds."""
    w = World(L, dtype, (8, 2, 64), 16, [150, 1], [400, 300])
    q = w.randn(151, w.Hq, w.D).mul_(2).to(w.t)
    out, lse, _ = attend(w, q, scale)
    o, l, to, tl, _ = reference(w, q, scale)
    close(out, o, to)
    close(lse, l, tl)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_prefix_that_sequences_share(L, dtype):
    w = World(L, dtype, (8, 2, 64), 16, [1, 40], [40, 90])
    w.tables[0] = w.tables[1][:2] + w.tables[0][2:]  # 32 common positions
    w.kv_lens[0] = 40
    q = w.randn(41, w.Hq, w.D).to(w.t)
    page, slot = w.at(w.tables[0], 40)
    w.k[page[32:], :, slot[32:]] = w.randn(8, 2, 64).to(w.t)
    w.v[page[32:], :, slot[32:]] = w.randn(8, 2, 64).to(w.t)
    out, _, batch = attend(w, q, 0.125)
    o, _, to, _, _ = reference(w, q, 0.125)
    close(out, o, to)
    with pytest.raises(L.LumenError) as e:  # whose weight would it be?
        L.paged_attention_mass(w.pool, batch, q.data_ptr(), 0.125, q.data_ptr())
    assert e.value.code == L._lib.ERR_INVALID


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [300, 5000]), ([20, 3, 1], [20, 64, 65]), ([200, 64], [700, 64])])
def test_positions_behind_a_token_do_not_reach_it(L, dtype, q_lens, kv_lens):
    """The same bits whether the positions behind a token hold large numbers or others."""
    w = World(L, dtype, (8, 2, 64), 16, q_lens, kv_lens)
    q = w.randn(sum(q_lens), w.Hq, w.D).to(w.t)
    first, lse, _ = attend(w, q, 0.125)
    for b, n in enumerate(q_lens):
        page, slot = w.at(w.tables[b], kv_lens[b])
        w.k[page[-1], :, slot[-1]] = 3e4 if dtype == "f32" else 2.0 ** 14
        w.v[page[-1], :, slot[-1]] = 1e30
    again, lse2, _ = attend(w, q, 0.125)
    last = torch.as_tensor(np.cumsum(q_lens) - 1)
    rest = torch.ones(sum(q_lens), dtype=torch.bool)
    rest[last] = False
    assert torch.equal(first[rest], again[rest]) and torch.equal(lse[rest], lse2[rest])


def test_the_same_bits_every_time(L):
    for dtype in ("bf16", "f32"):
        w = World(L, dtype, (32, 8, 128), 64, [1, 1, 100], [3000, 10, 900])
        q = w.randn(102, w.Hq, w.D).to(w.t)
        a, b = attend(w, q, 0.088), attend(w, q, 0.088)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ---- append -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads", [(8, 2, 64), (7, 1, 128), (5, 5, 64)], ids=str)
@pytest.mark.parametrize("norm,rope,odd", [(True, True, 0), (False, True, 1), (True, False, 3), (False, False, 0), (True, True, 2)])
def test_append(L, dtype, heads, norm, rope, odd):
    """`odd` floats between rows and in front of them: parts of a wider product at any alignment."""
    append_of(L, dtype, heads, norm, rope, odd, [1, 0, 37, 2], [1, 30, 100, 33], [900, 0, 5, 63])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,odd", [((8, 2, 64), 0), ((8, 2, 64), 4), ((7, 1, 128), 0), ((32, 8, 128), 0), ((48, 16, 128), 0), ((7, 1, 128), 2)], ids=str)
@pytest.mark.parametrize("norm,rope", [(True, True), (False, False)])
def test_append_of_many_tokens(L, dtype, heads, odd, norm, rope):
    """Enough for CTAs that stay and bring several tokens through each stage of their ring; rows too long for it, and rows at odd places."""
    append_of(L, dtype, heads, norm, rope, odd, [700, 1, 1300], [900, 33, 1300], [7, 1999, 0])


def append_of(L, dtype, heads, norm, rope, odd, q_lens, kv_lens, first):
    w = World(L, dtype, heads, 16, q_lens, kv_lens)
    T, D, n = sum(q_lens), w.D, w.Hq + 2 * w.Hkv
    flat = w.randn(T * (n * D + odd) + odd)
    x = flat[odd:].view(T, n * D + odd)[:, : n * D].reshape(T, n, D).double().cpu()
    angle = np.arange(2000)[:, None] * 10000.0 ** (-np.arange(0, D, 2) / D)
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    tables = L.RotaryEmbedding.from_tables(cos, sin) if rope else None
    gq, gk = 1 + 0.1 * w.randn(D), 1 + 0.1 * w.randn(D)
    before = [t.clone() for t in (w.k, w.v, w.mass)]
    batch = w.batch(first_pos=first)
    out = torch.full((T + 1, w.Hq, D), 77.0, dtype=w.t, device=DEV)
    torch.cuda.synchronize()
    at, row = flat.data_ptr() + 4 * odd, n * D + odd
    L.paged_append(w.pool, batch, at, at + 4 * w.Hq * D, at + 4 * (w.Hq + w.Hkv) * D, row, row, out.data_ptr(), rope=tables,
                   **(dict(q_norm_ptr=gq.data_ptr(), k_norm_ptr=gk.data_ptr(), eps=1e-5) if norm else {}))
    w.pool.ctx.synchronize()

    pos = np.concatenate([first[b] + np.arange(m) for b, m in enumerate(q_lens)])

    def heads_of(y, g):
        big = y.abs()
        if norm:
            inv = 1 / (y.square().mean(-1, keepdim=True) + 1e-5).sqrt()
            y, big = y * inv * g.double().cpu(), big * inv * g.double().cpu().abs()
        if rope:
            c, s = (torch.as_tensor(t[pos].astype(np.float64))[:, None] for t in (cos, sin))
            a, b = y[..., : D // 2], y[..., D // 2:]
            y = torch.cat([a * c - b * s, b * c + a * s], -1)
            a, b = big[..., : D // 2], big[..., D // 2:]
            big = torch.cat([a * c.abs() + b * s.abs(), b * c.abs() + a * s.abs()], -1)
        # norm: D roundings of the sum, halved by the root, and four more; rotation: three; then the type's own
        return y, big * ((D / 2 + 8) * 2.0 ** -23) + (y.abs() * 2.0 ** -8 if dtype == "bf16" else 0)

    q, tq = heads_of(x[:, : w.Hq], gq)
    close(out[:-1].double().cpu(), q, tq)
    assert (out[-1] == 77).all()
    k, tk = heads_of(x[:, w.Hq: w.Hq + w.Hkv], gk)
    v = x[:, w.Hq + w.Hkv:]
    t = 0
    for b, m in enumerate(q_lens):
        page, slot = (y[kv_lens[b] - m:] for y in w.at(w.tables[b], kv_lens[b]))
        close(w.k[page, :, slot].double().cpu(), k[t: t + m], tk[t: t + m])
        close(w.v[page, :, slot].double().cpu(), v[t: t + m].float().to(w.t).double(), torch.zeros_like(v[t: t + m]))
        assert not w.mass[page, :, slot].any()
        for now, then in zip((w.k, w.v, w.mass), before):  # everything else stays, NaN and all
            then[page, :, slot] = now[page, :, slot]
        t += m
    for now, then in zip((w.k, w.v, w.mass), before):
        assert torch.equal(now.nan_to_num(5.0, 6.0, 7.0), then.nan_to_num(5.0, 6.0, 7.0))


# ---- what the positions were looked at -------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads", [(8, 2, 64), (7, 1, 128), (32, 8, 128), (4, 4, 64)], ids=str)
@pytest.mark.parametrize("lens", [([1], [1]), ([1, 0, 1, 1], [64, 50, 129, 2047]), ([17, 300, 1], [17, 900, 65]), ([3, 0], [1000, 0])], ids=str)
@pytest.mark.parametrize("causal", [True, False])
def test_observed_weights(L, dtype, heads, lens, causal):
    q_lens, kv_lens = lens
    w = World(L, dtype, heads, 32, q_lens, kv_lens)
    q = w.randn(sum(q_lens), w.Hq, w.D).mul_(2).to(w.t)
    scale = w.D ** -0.5
    batch = w.batch(causal=causal)
    out, lse = torch.empty_like(q), torch.empty(sum(q_lens), w.Hq, device=DEV)
    before = w.mass.clone()
    torch.cuda.synchronize()
    for _ in range(2):
        L.paged_attention(w.pool, batch, q.data_ptr(), scale, out.data_ptr(), lse_ptr=lse.data_ptr())
        L.paged_attention_mass(w.pool, batch, q.data_ptr(), scale, lse.data_ptr())
    w.pool.ctx.synchronize()
    mass = reference(w, q, scale, causal)[4]
    for b, n in enumerate(q_lens):
        if n and kv_lens[b]:
            page, slot = w.at(w.tables[b], kv_lens[b])
            had = before[page, :, slot].double().cpu()
            gain, tol = mass[b]
            close(w.mass[page, :, slot].double().cpu(), had + 2 * gain, 2 * tol + (had + 2 * gain) * 2.0 ** -22)
            before[page, :, slot] = w.mass[page, :, slot]
    assert torch.equal(w.mass.nan_to_num(5.0), before.nan_to_num(5.0))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [8, 16, 17, 24, 25])
def test_observed_weights_by_every_kernel(L, dtype, d, n):
    """Four heads to a key head: 64 and 96 rows are the most that the kernel for few rows takes; long sequences are cut, the new tokens lie on a cut."""
    w = World(L, dtype, (8, 2, d), 16, [n, 1, n, 2], [3001, 40, n, 1024], seed=n)
    q = w.randn(2 * n + 3, w.Hq, w.D).mul_(2).to(w.t)
    scale = w.D ** -0.5
    _, lse, batch = attend(w, q, scale)
    lse = lse.float().to(DEV)
    before = w.mass.clone()
    torch.cuda.synchronize()
    L.paged_attention_mass(w.pool, batch, q.data_ptr(), scale, lse.data_ptr())
    w.pool.ctx.synchronize()
    mass = reference(w, q, scale)[4]
    for b, kv in enumerate(w.kv_lens):
        page, slot = w.at(w.tables[b], kv)
        had = before[page, :, slot].double().cpu()
        gain, tol = mass[b]
        close(w.mass[page, :, slot].double().cpu(), had + gain, tol + (had + gain) * 2.0 ** -22)
        before[page, :, slot] = w.mass[page, :, slot]
    assert torch.equal(w.mass.nan_to_num(5.0), before.nan_to_num(5.0))


def test_observed_weights_have_the_same_bits_every_time(L):
    for dtype in ("bf16", "f32"):
        got = []
        for _ in range(2):
            w = World(L, dtype, (32, 8, 128), 64, [1, 150], [3000, 900])
            q = w.randn(151, w.Hq, w.D).to(w.t)
            _, _, batch = attend(w, q, 0.088)
            lse = torch.zeros(151, w.Hq, device=DEV)
            torch.cuda.synchronize()
            L.paged_attention_mass(w.pool, batch, q.data_ptr(), 0.01, lse.data_ptr())
            w.pool.ctx.synchronize()
            got.append(w.mass.nan_to_num(5.0).clone())
        assert torch.equal(*got)


# ---- eviction -------------------------------------------------------------------------------------------------------
def _chosen(m, keep, recent):
    """Positions that stay, from the masses of one key head."""
    last = min(recent, keep)
    old = len(m) - last
    key = np.where(np.isnan(m[:old]), -np.inf, m[:old].astype(np.float64))
    nan = np.isnan(m[:old])
    order = np.lexsort((np.arange(old), -key, nan))[: keep - last]  # NaN below everything, -infinity too
    return np.sort(np.concatenate([order, np.arange(old, len(m))])).astype(np.int64)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads", [(8, 2, 64), (4, 1, 128)], ids=str)
@pytest.mark.parametrize("kv,keep,recent", [([1], [1], 0), ([1], [0], 3), ([64, 0, 3000, 65], [13, 0, 1500, 65], 16), ([5000], [4999], 0), ([2049, 300], [1, 200], 1000),
                                            ([1500, 40], [700, 39], 1), ([6000, 7, 0, 4500], [2000, 7, 0, 4499], 30)])
@pytest.mark.parametrize("kind", ["smooth", "ties", "wild"])
def test_evict(L, dtype, heads, kv, keep, recent, kind):
    w = World(L, dtype, heads, 32, [0] * len(kv), kv, extra=keep)
    for b, n in enumerate(kv):
        m = torch.rand(n, w.Hkv, generator=w.g, device=DEV)
        if kind == "ties":
            m = (m * 4).floor()
        if kind == "wild":
            m = torch.where(m < 0.2, float("nan"), torch.where(m < 0.3, float("inf"), torch.where(m < 0.4, -float("inf"), torch.where(m < 0.5, -0.0, torch.where(m < 0.6, 0.0, m - 0.8)))))
        w.put(w.mass, b, m)
    a, z = w.batch(), w.batch(q_lens=[0] * len(kv), kv_lens=keep, tables=w.extra_tables)
    stride = max(keep) + 3
    kept = torch.full((len(kv), w.Hkv, stride), -7, dtype=torch.int32, device=DEV)
    want = [t.clone() for t in (w.k, w.v, w.mass)]
    for b, n in enumerate(kv):
        for h in range(w.Hkv):
            stay = _chosen(w.rows(w.mass, w.tables[b], n)[:, h].cpu().numpy(), keep[b], recent)
            sp, ss = (y[stay] for y in w.at(w.tables[b], n))
            dp, ds = w.at(w.extra_tables[b], keep[b])
            for t in want:
                t[dp, h, ds] = t[sp, h, ss]
    torch.cuda.synchronize()
    L.paged_evict(w.pool, a, z, recent, kept.data_ptr(), stride)
    w.pool.ctx.synchronize()
    for b, n in enumerate(kv):
        for h in range(w.Hkv):
            stay = _chosen(w.rows(w.mass, w.tables[b], n)[:, h].cpu().numpy(), keep[b], recent)
            assert kept[b, h, : keep[b]].tolist() == stay.tolist() and (kept[b, h, keep[b]:] == -7).all()
    for got, t in zip((w.k, w.v, w.mass), want):
        assert torch.equal(got.nan_to_num(5.0, 6.0, 7.0), t.nan_to_num(5.0, 6.0, 7.0))


@pytest.mark.parametrize("n", [4096, 4097, 45000, 333000])
@pytest.mark.parametrize("keep", [900, 4000])
def test_evict_from_long_caches(L, n, keep):
    """By one SM, by several, and too long for their shared memory."""
    w = World(L, "f32", (4, 2, 64), 256, [0, 0], [n, 100], extra=[keep, 100])
    w.put(w.mass, 0, (torch.rand(n, 2, generator=w.g, device=DEV) * 5000).floor())
    kept = torch.full((2, 2, keep), -7, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    L.paged_evict(w.pool, w.batch(), w.batch(kv_lens=[keep, 100], tables=w.extra_tables), 100, kept.data_ptr(), keep)
    w.pool.ctx.synchronize()
    m = w.rows(w.mass, w.tables[0], n).cpu().numpy()
    for h in range(2):
        stay = _chosen(m[:, h], keep, 100)
        assert kept[0, h].tolist() == stay.tolist() and kept[1, h, :100].tolist() == list(range(100))
        assert torch.equal(w.rows(w.v, w.extra_tables[0], keep)[:, h], w.rows(w.v, w.tables[0], n)[torch.as_tensor(stay, device=DEV), h])


# ---- refusals ------------------------------------------------------------------------------------------------------
def test_refusals(L, ctx):
    def refused(code, call, *a, **k):
        with pytest.raises(L.LumenError) as e:
            call(*a, **k)
        assert e.value.code == getattr(L._lib, code), e.value

    for args, code in [((4, 12, 2, 64), "ERR_UNSUPPORTED"), ((4, 4, 2, 64), "ERR_UNSUPPORTED"), ((4, 512, 2, 64), "ERR_UNSUPPORTED"), ((4, 16, 2, 80), "ERR_UNSUPPORTED"),
                       ((0, 16, 2, 64), "ERR_INVALID"), ((4, 16, 0, 64), "ERR_INVALID"), ((2 ** 40, 16, 2, 64), "ERR_INVALID"), ((2 ** 26, 16, 1024, 128), "ERR_CUDA")]:
        refused(code, L.PagePool, *args)
    refused("ERR_DTYPE", L.PagePool, 4, 16, 2, 64, 7)
    pool, other, f32 = L.PagePool(8, 16, 2, 64), L.PagePool(9, 16, 2, 64), L.PagePool(8, 16, 2, 64, L.F32)
    for q, kv, tables, code in [([1], [17], [[0]], "ERR_KV_OVERFLOW"), ([1, 1], [17, 17], [[0], [1, 2]], "ERR_INVALID"), ([1], [17], np.zeros((1, 1), int), "ERR_KV_OVERFLOW"), ([1], [17], [[0, 8]], "ERR_INVALID"), ([1], [17], [[3, 3]], "ERR_INVALID"),
                                ([2], [1], [[0]], "ERR_SHAPE"), ([-1], [1], [[0]], "ERR_INVALID"), ([1, 1], [1], [[0], [1]], "ERR_SHAPE"), ([1], [1], [[0], [1]], "ERR_SHAPE"),
                                ([1.5], [2], [[0]], "ERR_INVALID"), ([1], [2 ** 31], [[0]], "ERR_INVALID")]:
        refused(code, L.PageBatch, pool, 4, q, kv, tables)
    refused("ERR_SHAPE", L.PageBatch, pool, 3, [1], [1], [[0]])
    refused("ERR_UNSUPPORTED", L.PageBatch, pool, 2 * 129, [1], [1], [[0]])
    refused("ERR_INVALID", L.PageBatch, pool, 4, [1], [1], [[0]], first_pos=[-1])

    batch = L.PageBatch(pool, 4, [1], [17], [[0, 1]])
    x = torch.zeros(4096, device=DEV)
    p = x.data_ptr()
    rope = L.RotaryEmbedding(64, 16, 10000.0)
    app = lambda b, **k: L.paged_append(**{**dict(pool=pool, batch=b, q_ptr=p, k_ptr=p, v_ptr=p, q_stride=256, kv_stride=128, q_out_ptr=p + 8192), **k})  # noqa: E731
    refused("ERR_SHAPE", app, batch, q_stride=255)
    refused("ERR_SHAPE", app, batch, kv_stride=127)
    refused("ERR_INVALID", app, batch, q_out_ptr=p + 8)
    refused("ERR_INVALID", app, batch, q_ptr=0)
    refused("ERR_INVALID", app, batch, q_out_ptr=p + 1008)  # (rows of 1024 bytes)
    refused("ERR_INVALID", app, batch, q_ptr=p + 4096, q_out_ptr=p)
    refused("ERR_ROPE_RANGE", app, batch, rope=rope)  # position 16 of 16
    refused("ERR_SHAPE", app, batch, rope=L.RotaryEmbedding(32, 99, 10000.0))
    refused("ERR_SHAPE", app, L.PageBatch(pool, 4, [3], [1], [[0]], causal=False))
    refused("ERR_INVALID", app, L.PageBatch(pool, 4, [1, 1], [16, 20], [[0], [0, 1]]))
    refused("ERR_SHAPE", app, batch, pool=other)
    att = lambda **k: L.paged_attention(**{**dict(pool=pool, batch=batch, q_ptr=p, scale=1.0, out_ptr=p + 8192), **k})  # noqa: E731
    refused("ERR_SHAPE", att, pool=f32)
    refused("ERR_INVALID", att, out_ptr=0)
    refused("ERR_INVALID", att, out_ptr=p + 8)
    refused("ERR_INVALID", att, out_ptr=p + 16)  # overlaps
    refused("ERR_INVALID", att, lse_ptr=p + 8192)
    refused("ERR_INVALID", att, lse_ptr=p + 508)
    refused("ERR_INVALID", att, scale=float("nan"))
    refused("ERR_INVALID", att, scale=float("inf"))
    refused("ERR_DTYPE", att, out_dtype=7)
    refused("ERR_DTYPE", att, pool=f32, batch=L.PageBatch(f32, 4, [1], [17], [[0, 1]]), out_dtype=L.BF16)
    refused("ERR_INVALID", L.paged_attention_mass, pool, batch, p, 1.0, 0)
    refused("ERR_SHAPE", L.paged_attention_mass, other, batch, p, 1.0, p)
    ev = lambda goal, stride=16, kept=p: L.paged_evict(pool, batch, goal, 0, kept, stride)  # noqa: E731
    goal = lambda n, t: L.PageBatch(pool, 4, [0] * len(n), n, t)  # noqa: E731
    refused("ERR_INVALID", ev, goal([10], [[1]]))
    refused("ERR_SHAPE", ev, goal([18], [[2, 3]]), 32)
    refused("ERR_SHAPE", ev, goal([10], [[2]]), 9)
    refused("ERR_SHAPE", ev, goal([10, 0], [[2], []]))
    refused("ERR_INVALID", ev, goal([10], [[2]]), 16, 0)
    two = L.PageBatch(pool, 4, [0, 0], [17, 17], [[0, 1], [0, 1]])
    refused("ERR_INVALID", L.paged_evict, pool, two, goal([10, 10], [[2], [2]]), 0, p, 16)
    refused("ERR_SHAPE", L.RotaryEmbedding.from_tables, np.zeros((4, 8)), np.zeros((4, 9)))
    lib = L._lib.load()
    for call in (lib.lumen_page_pool_free, lib.lumen_page_batch_free):
        assert call(None) == L._lib.ERR_INVALID
    torch.cuda.synchronize()
    ctx.synchronize()


def test_refusals_of_the_pool_s_own_memory(L, ctx):
    """Rows and results may not lie in the pool; scales that overflow with log2(e) are refused; nothing is freed into a graph."""
    def refused(call, *a, **k):
        with pytest.raises(L.LumenError) as e:
            call(*a, **k)
        assert e.value.code == L._lib.ERR_INVALID, e.value

    pool = L.PagePool(8, 16, 2, 64, L.F32)
    batch, goal = L.PageBatch(pool, 4, [1], [17], [[0, 1]]), L.PageBatch(pool, 4, [0], [10], [[2]])
    x = torch.zeros(4096, device=DEV)
    p, last = x.data_ptr(), pool.mass_ptr + 8 * 2 * 16 * 4 - 16  # (the pool's last 16 bytes)
    row = dict(pool=pool, batch=batch, q_ptr=p, k_ptr=p, v_ptr=p, q_stride=256, kv_stride=128, q_out_ptr=p + 8192)
    for at in (pool.k_ptr, pool.v_ptr, pool.mass_ptr, last):
        for name in ("q_ptr", "k_ptr", "v_ptr", "q_out_ptr"):
            refused(L.paged_append, **{**row, name: at})
        refused(L.paged_attention, pool, batch, p, 1.0, at)
        refused(L.paged_attention, pool, batch, p, 1.0, p + 8192, lse_ptr=at)
        refused(L.paged_evict, pool, batch, goal, 0, at, 16)
    for scale in (2.0 ** 127, -(2.0 ** 127)):
        refused(L.paged_attention, pool, batch, p, scale, p + 8192)
        refused(L.paged_attention_mass, pool, batch, p, scale, p)
    L.paged_attention(pool, batch, p, 2.0 ** 126, p + 8192)
    lib, other, spare = L._lib.load(), L.PageBatch(pool, 4, [1], [1], [[0]]), L.PagePool(1, 16, 1, 64)
    ctx.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.ExternalStream(ctx.stream)):
        L.paged_attention(pool, batch, p, 1.0, p + 8192)
        refused(L.PagePool, 1, 16, 1, 64)
        assert lib.lumen_page_batch_free(other.h) == lib.lumen_page_pool_free(spare.h) == L._lib.ERR_INVALID
    L.paged_attention(pool, other, p, 1.0, p + 8192)  # (still there)
    L.paged_append(**{**row, "pool": spare, "batch": L.PageBatch(spare, 1, [1], [1], [[0]])})
    ctx.synchronize()


def test_nothing_to_do(L):
    """No sequences, no new tokens, nothing to keep: accepted, and nothing is written."""
    pool = L.PagePool(8, 16, 2, 64)
    x = torch.full((4096,), 3.0, device=DEV)
    kept = torch.full((64,), -1, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    p = x.data_ptr()
    before = pool.ctx.launch_count
    for batch in (L.PageBatch(pool, 4, [], [], []), L.PageBatch(pool, 4, [0, 0], [17, 0], [[0, 1], []])):
        L.paged_append(pool, batch, p, p, p, 256, 128, p)
        L.paged_attention(pool, batch, p, 1.0, p + 8192, lse_ptr=p)
        L.paged_attention_mass(pool, batch, p, 1.0, p)
        L.paged_evict(pool, batch, L.PageBatch(pool, 4, [0] * len(batch.q_lens), [0] * len(batch.q_lens), [[]] * len(batch.q_lens)), 4, kept.data_ptr(), 0)
    pool.ctx.synchronize()
    assert pool.ctx.launch_count == before and (x == 3).all() and (kept == -1).all()


def test_a_batch_fits_the_pools_of_all_layers(L):
    w, other = World(L, "bf16", (8, 2, 64), 16, [1, 40], [100, 90]), World(L, "bf16", (8, 2, 64), 16, [1, 40], [100, 90], seed=0)
    other.k.copy_(w.k.flip(0))
    other.v.copy_(w.v.flip(0))
    other.tables = [[w.pages - 1 - t for t in table] for table in w.tables]
    q = w.randn(41, 8, 64).to(w.t)
    a, b = attend(w, q, 0.125), attend(other, q, 0.125)
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    L.paged_attention(other.pool, b[2], q.data_ptr(), 0.125, out.data_ptr())
    L.paged_attention(w.pool, a[2], q.data_ptr(), 0.125, out.data_ptr())
    L.paged_attention(other.pool, L.PageBatch(w.pool, 8, [1, 40], [100, 90], other.tables), q.data_ptr(), 0.125, out.data_ptr())
    w.pool.ctx.synchronize()
    assert torch.equal(out.double().cpu(), a[0]) and torch.equal(a[0], b[0])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_more_sequences_than_a_grid_has_rows(L, dtype):
    """33000 short sequences: one token each to 2 positions, observed, then one of them stays."""
    n, D = 33000, 64
    w = World(L, dtype, (2, 1, D), 8, [], [], spare=2 * n)
    w.k.copy_(w.randn(2 * n, 1, 8, D))
    w.v.copy_(w.randn(2 * n, 1, 8, D))
    w.mass.zero_()
    tables = np.random.default_rng(1).permutation(2 * n)
    batch, goal = w.batch(q_lens=[1] * n, kv_lens=[2] * n, tables=tables[:n, None]), w.batch(q_lens=[0] * n, kv_lens=[1] * n, tables=tables[n:, None])
    q = w.randn(n, 2, D).to(w.t)
    out, lse, kept = torch.empty_like(q), torch.empty(n, 2, device=DEV), torch.full((n, 1), -7, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    L.paged_attention(w.pool, batch, q.data_ptr(), 0.3, out.data_ptr(), lse_ptr=lse.data_ptr())
    L.paged_attention_mass(w.pool, batch, q.data_ptr(), 0.3, lse.data_ptr())
    L.paged_evict(w.pool, batch, goal, 0, kept.data_ptr(), 1)
    w.pool.ctx.synchronize()
    at = torch.as_tensor(tables, device=DEV)
    k, v = (x[at[:n], 0, :2].double() for x in (w.k, w.v))
    p = torch.softmax(torch.einsum("nhd,njd->nhj", q.double(), k) * 0.3, -1)
    big = torch.einsum("nhd,njd->nhj", q.double().abs(), k.abs()).amax(-1, keepdim=True) * 0.3
    rel = 2 * (D + 4) * 2.0 ** -23 * big + 2.0 ** -19 + (2 ** -8 if dtype == "bf16" else 0)
    o = torch.einsum("nhj,njd->nhd", p, v)
    close(out.double().cpu(), o.cpu(), (2 * rel * torch.einsum("nhj,njd->nhd", p, v.abs()) + o.abs() * (2.0 ** -8 if dtype == "bf16" else 0)).cpu())
    gain = p.sum(1)
    got = w.mass[at[:n], 0, :2].double()
    close(got.cpu(), gain.cpu(), (2 * rel.amax(1) * gain + 1e-6).cpu())
    want = (got[:, 1] > got[:, 0]).int()
    assert torch.equal(kept[:, 0], want)
    assert torch.equal(w.v[at[n:], 0, 0], w.v[at[:n]][torch.arange(n, device=DEV), 0, want.long()])


# ---- captured, and together ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_captured_steps(L, ctx, dtype):
    """Two batches of two captured graphs, replayed in turn with new inputs; a batch is not made while its stream is captured."""
    w = World(L, dtype, (8, 2, 128), 64, [1, 130], [3001, 600])
    w2 = World(L, dtype, (8, 2, 128), 64, [2], [4000], seed=5)
    stream = torch.cuda.ExternalStream(ctx.stream)
    made = []
    for x in (w, w2):
        n = sum(x.q_lens)
        s = dict(w=x, batch=x.batch(), q=torch.zeros(n, 8, 128, dtype=x.t, device=DEV), out=torch.zeros(n, 8, 128, dtype=x.t, device=DEV), lse=torch.zeros(n, 8, device=DEV))
        call = lambda s=s: (L.paged_attention(s["w"].pool, s["batch"], s["q"].data_ptr(), 0.1, s["out"].data_ptr(), lse_ptr=s["lse"].data_ptr()),  # noqa: E731
                            L.paged_attention_mass(s["w"].pool, s["batch"], s["q"].data_ptr(), 0.1, s["lse"].data_ptr()))
        torch.cuda.synchronize()
        call()
        ctx.synchronize()
        s["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(s["graph"], stream=stream):
            call()
            with pytest.raises(L.LumenError) as e:
                x.batch()
            assert e.value.code == L._lib.ERR_INVALID
        made.append(s)
    for turn in range(3):
        for s in made:
            s["q"].copy_(s["w"].randn(*s["q"].shape))
        torch.cuda.synchronize()
        before = [s["w"].mass.clone() for s in made]
        with torch.cuda.stream(stream):
            for s in made:
                s["graph"].replay()
        torch.cuda.synchronize()
        for s, m in zip(made, before):
            o, l, to, tl, gain = reference(s["w"], s["q"], 0.1)
            close(s["out"].double().cpu(), o, to)
            close(s["lse"].double().cpu(), l, tl)
            for b, n in enumerate(s["w"].kv_lens):
                had = s["w"].rows(m, s["w"].tables[b], n).double().cpu()
                close(s["w"].rows(s["w"].mass, s["w"].tables[b], n).double().cpu(), had + gain[b][0], gain[b][1] + (had + gain[b][0]) * 2.0 ** -22)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_conversation(L, dtype):
    """Two sequences: prompts in chunks, single tokens, the weights observed all along; then one cache shrinks to a third and its sequence goes on,
    its positions counted from what it has read.  Every step against a plain cache of lists."""
    w = World(L, dtype, (8, 2, 64), 16, [0, 0], [0, 0], spare=64)
    D, Hq, Hkv, G, scale = 64, 8, 2, 4, 0.125
    free = list(range(w.pages))
    tables = [[], []]
    cache = [dict(k=torch.zeros(0, Hkv, D, dtype=torch.float64), v=torch.zeros(0, Hkv, D, dtype=torch.float64), m=torch.zeros(0, Hkv, dtype=torch.float64)) for _ in range(2)]
    angle = np.arange(2000)[:, None] * 10000.0 ** (-np.arange(0, D, 2) / D)
    rope = L.RotaryEmbedding.from_tables(np.cos(angle), np.sin(angle))
    gain = 1 + 0.1 * w.randn(D)
    read = [0, 0]
    eps = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -22

    def step(news):
        lens = [c["k"].shape[0] + n for c, n in zip(cache, news)]
        for b in range(2):
            while len(tables[b]) * 16 < lens[b]:
                tables[b].append(free.pop())
        batch = w.batch(q_lens=news, kv_lens=lens, tables=tables, first_pos=read)
        T = sum(news)
        qkv = w.randn(T, (Hq + 2 * Hkv) * D)
        q, out, lse = torch.empty(T, Hq, D, dtype=w.t, device=DEV), torch.empty(T, Hq, D, dtype=w.t, device=DEV), torch.empty(T, Hq, device=DEV)
        torch.cuda.synchronize()
        at, row = qkv.data_ptr(), qkv.shape[1]
        L.paged_append(w.pool, batch, at, at + 4 * Hq * D, at + 4 * (Hq + Hkv) * D, row, row, q.data_ptr(), rope=rope, q_norm_ptr=gain.data_ptr(), k_norm_ptr=gain.data_ptr(), eps=1e-6)
        L.paged_attention(w.pool, batch, q.data_ptr(), scale, out.data_ptr(), lse_ptr=lse.data_ptr())
        L.paged_attention_mass(w.pool, batch, q.data_ptr(), scale, lse.data_ptr())
        w.pool.ctx.synchronize()
        t = 0
        for b, n in enumerate(news):
            x = qkv[t: t + n].double().cpu().view(n, Hq + 2 * Hkv, D)
            pos = read[b] + np.arange(n)

            def head(y):
                y = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * gain.double().cpu()
                c, s = torch.as_tensor(np.cos(angle[pos]))[:, None], torch.as_tensor(np.sin(angle[pos]))[:, None]
                return torch.cat([y[..., :32] * c - y[..., 32:] * s, y[..., 32:] * c + y[..., :32] * s], -1)

            c = cache[b]
            # what was rounded on the way into the cache is taken from it: this test is about what meets what
            newk, newq = head(x[:, Hq: Hq + Hkv]), head(x[:, :Hq])
            c["k"], c["v"] = torch.cat([c["k"], newk]), torch.cat([c["v"], x[:, Hq + Hkv:]])
            c["m"] = torch.cat([c["m"], torch.zeros(n, Hkv, dtype=torch.float64)])
            total = c["k"].shape[0]
            have = w.rows(w.k, tables[b], total).double().cpu()
            # (a norm of 64 numbers and a rotation in 32 bits, then one rounding)
            assert ((have - c["k"]).abs() <= c["k"].abs() * eps + 64 * 2.0 ** -22).all()
            c["k"], c["v"] = have, w.rows(w.v, tables[b], total).double().cpu()
            gq = q[t: t + n].double().cpu()
            assert ((gq - newq).abs() <= newq.abs() * eps + 64 * 2.0 ** -22).all()
            s = torch.einsum("thd,jhd->htj", gq, c["k"].repeat_interleave(G, 1)) * scale
            s = s.masked_fill(torch.arange(total)[None] > total - n + torch.arange(n)[:, None], -np.inf)
            p = torch.softmax(s, -1)
            o = torch.einsum("htj,jhd->thd", p, c["v"].repeat_interleave(G, 1))
            most = float(c["v"].abs().max())
            assert ((out[t: t + n].double().cpu() - o).abs() <= most * (2 * eps + 1e-5)).all()
            c["m"] = c["m"] + p.view(Hkv, G, n, total).sum((1, 2)).T
            got = w.rows(w.mass, tables[b], total).double().cpu()
            assert ((got - c["m"]).abs() <= 1e-4 * c["m"] + 1e-5).all()
            c["m"] = got
            read[b] += n
            t += n

    step([100, 17])
    step([150, 1])
    for _ in range(3):
        step([1, 1])
    step([0, 40])
    total, keep, recent = cache[0]["k"].shape[0], 84, 20
    goal = [free.pop() for _ in range(-(-keep // 16))]
    kept = torch.zeros(1, Hkv, keep, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    L.paged_evict(w.pool, w.batch(q_lens=[0], kv_lens=[total], tables=[tables[0]]), w.batch(q_lens=[0], kv_lens=[keep], tables=[goal]), recent, kept.data_ptr(), keep)
    w.pool.ctx.synchronize()
    c = cache[0]
    stay = [torch.as_tensor(_chosen(c["m"][:, h].numpy(), keep, recent)) for h in range(Hkv)]
    assert kept[0].tolist() == [s.tolist() for s in stay]
    for name in ("k", "v", "m"):
        c[name] = torch.stack([c[name][s, h] for h, s in enumerate(stay)], 1)
    free += tables[0]
    tables[0] = goal
    step([1, 1])
    step([70, 0])
    step([1, 1])
