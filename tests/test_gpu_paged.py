"""Paged KV cache on the GPU through the C ABI: append, attention and eviction against plain 64-bit
implementations.

Tolerances.  u = 2^-23 covers rounding to nearest (2^-24) and truncating accumulators.  By the probabilistic
rounding-error bound (Higham and Mary, 2019), a sum of n products errs by at most 8 sqrt(n) u of the sum of
their magnitudes, except with a probability far below any test's.  A score therefore errs by
ds = 8 sqrt(D) u scale sum|q k|, a softmax weight by a relative 2 ds + 8 sqrt(n) u + 8 u, and an output by that
(plus 8 sqrt(n) u for its own sum) times sum p |V|."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -23
HALF_ULP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
KV = {"f32": 0, "f16": 1, "bf16": 2}


class Cache:
    """One layer's pool, its page table and a shuffled page order (numpy mirrors are built from the device)."""

    def __init__(self, torch, kv, n_head, n_head_kv, dim, page, lens, cols=None, seed=0, split=False, mass=True,
                 spare=2, pool_fill=None):
        from mcpm import engine as E
        self.torch, self.E, self.kv, self.page, self.lens = torch, E, kv, page, list(lens)
        self.n_head, self.n_head_kv, self.dim = n_head, n_head_kv, dim
        rng = np.random.default_rng(seed)
        self.rng = rng
        want = [-(-n // page) for n in lens]
        self.cols = cols or max(1, max(want))
        self.n_pages = sum(want) + spare
        order = rng.permutation(self.n_pages).astype(np.int32)
        self.free = list(order[sum(want):])
        self.table = np.full((len(lens), self.cols), -1, np.int32)
        at = 0
        for i, w in enumerate(want):
            self.table[i, :w] = order[at:at + w]
            at += w
        dt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kv]
        shape = (self.n_pages, n_head_kv, page, dim) if split else (self.n_pages, page, n_head_kv, dim)

        def pool():
            x = rng.normal(0, 1, shape).astype(np.float32) if pool_fill is None else np.full(shape, pool_fill, np.float32)
            x = torch.from_numpy(x).to(dt).cuda()
            return x.transpose(1, 2) if split else x

        self.k, self.v = pool(), pool()
        self.mass = torch.from_numpy(rng.exponential(0.5, (self.n_pages, n_head_kv, page)).astype(np.float32)).cuda() if mass else None
        self.make(len(lens))

    def make(self, max_seqs):
        E, k = self.E, self.k
        self.cfg = E.paged_config(KV[self.kv], self.n_head, self.n_head_kv, self.dim, self.page, self.n_pages, max_seqs,
                                  self.cols, k.stride(0), k.stride(1), k.stride(2))
        self.pool = E.paged_pool(k.data_ptr(), self.v.data_ptr(), self.mass.data_ptr() if self.mass is not None else 0)
        self.ws = self.torch.zeros(E.paged_workspace_bytes(self.cfg), dtype=self.torch.uint8, device="cuda")

    def dev(self, a):
        return self.torch.from_numpy(np.ascontiguousarray(a)).cuda()

    def places(self, seq, n=None, table=None):
        """Present positions of a sequence and their pages and slots."""
        row = (self.table if table is None else table)[seq]
        j = np.arange(min(max(0, self.lens[seq] if n is None else n), self.cols * self.page))
        p = row[j // self.page]
        ok = (p >= 0) & (p < self.n_pages)
        return j[ok], p[ok], (j % self.page)[ok]

    def host(self):
        return self.k.double().cpu().numpy(), self.v.double().cpu().numpy()

    def attend(self, q, scale=0.0, out=None, stream=0, lens=None):
        torch = self.torch
        n = len(self.lens)
        self.t_dev, self.l_dev = self.dev(self.table), self.dev(np.array(self.lens if lens is None else lens, np.int32))
        out = torch.full((n, self.n_head * self.dim), 7.0, device="cuda") if out is None else out
        self.E.paged_attention(self.cfg, self.pool, self.t_dev.data_ptr(), self.l_dev.data_ptr(), n, q.data_ptr(),
                               out.data_ptr(), self.ws.data_ptr(), self.ws.numel(), q_stride=q.stride(0), scale=scale, stream=stream)
        torch.cuda.synchronize()
        return out


def expected_attention(c, q, scale):
    """(out, out tolerance, {(page, head, slot): (weight, tolerance)}) in 64 bits."""
    k, v = c.host()
    n, g = len(c.lens), c.n_head // c.n_head_kv
    qq = q.double().cpu().numpy().reshape(n, c.n_head, c.dim)
    out = np.zeros((n, c.n_head, c.dim))
    tol = np.zeros_like(out)
    add, add_tol = np.zeros((c.n_pages, c.n_head_kv, c.page)), np.zeros((c.n_pages, c.n_head_kv, c.page))
    for i in range(n):
        j, p, s = c.places(i)
        if not j.size:
            continue
        for h in range(c.n_head):
            kk, vv = k[p, s, h // g], v[p, s, h // g]
            score = scale * kk @ qq[i, h]
            ds = 8 * np.sqrt(c.dim) * U * scale * (np.abs(kk) @ np.abs(qq[i, h])).max()
            e = np.exp(score - score.max())
            w = e / e.sum()
            rel = 2 * ds + 8 * np.sqrt(j.size) * U + 8 * U
            out[i, h] = w @ vv
            tol[i, h] = (rel + 8 * np.sqrt(j.size) * U) * (w @ np.abs(vv)) + 1e-30
            add[p, h // g, s] += w
            add_tol[p, h // g, s] += rel * w
    return out.reshape(n, -1), tol.reshape(n, -1), add, add_tol


def check_attention(c, q, scale=0.0):
    before = c.mass.double().cpu().numpy() if c.mass is not None else None
    want, tol, add, add_tol = expected_attention(c, q, scale or c.dim ** -0.5)
    got = c.attend(q, scale).double().cpu().numpy()
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / tol)
    if before is not None:
        m = c.mass.double().cpu().numpy()
        lim = add_tol + 2 * U * (before + add)
        assert np.all(np.abs(m - before - add) <= lim), np.max(np.abs(m - before - add) - lim)
        assert np.array_equal(m[add == 0], before[add == 0])   # nothing else is touched
    return got


HEADS = [(16, 2, 128), (12, 4, 64), (8, 8, 64), (16, 1, 128), (20, 4, 128), (9, 3, 64), (1, 1, 128)]


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_head,n_head_kv,dim", HEADS)
def test_attention_heads_and_types(cuda, kv, n_head, n_head_kv, dim):
    c = Cache(cuda, kv, n_head, n_head_kv, dim, 16, [1, 0, 15, 16, 17, 63, 64, 65, 333, 1025], seed=n_head * 7 + dim)
    check_attention(c, 1.5 * cuda.randn(10, n_head * dim, device="cuda"))


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page,split", [(1, False), (7, True), (24, False), (64, True), (100, False), (1000, True)])
def test_attention_pages_and_strides(cuda, kv, page, split):
    c = Cache(cuda, kv, 16, 2, 128, page, [1, 2, 7, 129, 500, 1001, 2049], seed=page, split=split, cols=2100 if page == 1 else None)
    wide = cuda.randn(7, 16 * 128 + 512, device="cuda")   # rows inside a wider projection
    check_attention(c, wide[:, :2048])


@pytest.mark.parametrize("kv", ["f32", "f16"])
def test_attention_absent_pages_and_empty_rows(cuda, kv):
    c = Cache(cuda, kv, 16, 2, 128, 16, [200, 0, 333, 16, 64, 700], seed=5)
    c.table[0, 3] = -1                  # a page in the middle
    c.table[2, 0] = c.n_pages           # ids beyond the pool are absent too
    c.table[2, 20] = 2 ** 31 - 1
    c.table[3, :] = -1                  # nothing left
    c.table[4, :3] = -2 ** 31           # all but the last page
    got = check_attention(c, cuda.randn(6, 2048, device="cuda"))
    assert not got[1].any() and not got[3].any()


def test_attention_lengths_are_clamped(cuda):
    c = Cache(cuda, "f16", 16, 2, 128, 16, [64, 64, 64], seed=6, mass=False)
    q = cuda.randn(3, 2048, device="cuda")
    want = c.attend(q, lens=[64, 0, 64])
    got = c.attend(q, lens=[2 ** 31 - 1, -2 ** 31, 64 + 1])   # more than the table has room for, and fewer than none
    assert cuda.equal(got, want) and not got[1].any()


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
def test_attention_ignores_what_is_not_visible(cuda, kv):
    """NaN, infinities and the type's extremes beyond the length and in absent pages change nothing."""
    c = Cache(cuda, kv, 16, 2, 128, 16, [35, 100, 5], seed=8, mass=False)
    c.table[1, 2] = -1
    q = cuda.randn(3, 2048, device="cuda")
    want = c.attend(q).clone()
    dirty = cuda.ones(c.n_pages, 16, dtype=cuda.bool, device="cuda")
    for i in range(3):
        _, p, s = c.places(i)
        dirty[c.dev(p).long(), c.dev(s).long()] = False
    for bad in (float("nan"), float("inf"), cuda.finfo(c.k.dtype).min):
        c.k[dirty] = bad
        c.v[dirty] = bad
        assert cuda.equal(c.attend(q), want)


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
def test_attention_large_and_equal_scores(cuda, kv):
    """Scores of +-10^4 (one weight takes all) and all-equal scores (the mean of V)."""
    c = Cache(cuda, kv, 16, 2, 128, 16, [300, 77], seed=9, mass=False)
    q = 1000.0 * cuda.randn(2, 2048, device="cuda")
    want, tol, _, _ = expected_attention(c, q, 128 ** -0.5)
    k, v = c.host()
    got = c.attend(q).double().cpu().numpy().reshape(2, 16, 128)
    assert np.all(np.isfinite(got))
    for i in range(2):
        j, p, s = c.places(i)
        for h in range(16):
            sc = k[p, s, h // 8] @ q[i].double().cpu().numpy().reshape(16, 128)[h] * 128 ** -0.5
            top = np.sort(sc)
            if top[-1] - top[-2] > 40:   # the rest weigh less than e^-40 < 2^-57
                assert np.allclose(got[i, h], v[p, s, h // 8][sc.argmax()], rtol=8 * U, atol=8 * U)
    zero = cuda.zeros(2, 2048, device="cuda")
    want, tol, _, _ = expected_attention(c, zero, 128 ** -0.5)
    got = c.attend(zero).double().cpu().numpy()
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e6, 1e20])
def test_attention_query_magnitudes(cuda, kv, size):
    """Queries far from unit size, with the scale that makes the scores ordinary."""
    c = Cache(cuda, kv, 16, 2, 128, 16, [200, 9], seed=10, mass=False)
    q = size * cuda.randn(2, 2048, device="cuda")
    want, tol, _, _ = expected_attention(c, q, 0.1 / size)
    got = c.attend(q, scale=0.1 / size).double().cpu().numpy()
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / tol)


@pytest.mark.parametrize("kv", ["f32", "bf16"])
@pytest.mark.parametrize("k_size,v_size", [(1e37, 1.0), (1.0, 1e36), (3e37, 3e36), (1e-20, 1e-15), (1e37, 1e-15)])
def test_attention_cache_magnitudes(cuda, kv, k_size, v_size):
    """K and V up to the ends of their types' range, with queries and a scale that make the scores ordinary.  At most
    7 x 3e36 x 12: sums over the 12 positions stay in range."""
    c = Cache(cuda, kv, 16, 2, 128, 16, [12, 9], seed=41, mass=False)
    c.k *= k_size
    c.v *= v_size
    assert bool(cuda.isfinite(c.k).all() & cuda.isfinite(c.v).all())
    for q_size in (1e-12, 1.0):
        q = q_size * cuda.randn(2, 2048, device="cuda")
        scale = float(np.float32(0.1 / q_size / k_size))
        want, tol, _, _ = expected_attention(c, q, scale)
        got = c.attend(q, scale=scale).double().cpu().numpy()
        assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / tol)


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
def test_attention_type_extremes(cuda, kv):
    """The type's largest value in every element of K, of either sign by position: scores of fp32's size or beyond give
    the positive positions all the weight; V at the largest value that a mean of 40 leaves in range."""
    c = Cache(cuda, kv, 16, 2, 128, 16, [40, 5], seed=42, mass=False)
    top = cuda.finfo(c.k.dtype).max
    want = []
    for i in range(2):
        j, p, s = c.places(i)
        sign = np.where(j % 3 == 1, 1.0, -1.0)
        c.k[c.dev(p).long(), c.dev(s).long()] = (c.dev(sign)[:, None, None] * top).to(c.k.dtype)
        want.append(c.v[c.dev(p[sign > 0]).long(), c.dev(s[sign > 0]).long()].double().mean(0))
    q = cuda.full((2, 2048), 2.0 ** -3, device="cuda")
    got = c.attend(q, scale=2.0 ** -5).double().view(2, 2, 8, 128)   # scores of +-top / 2: 128 * 2^-8 of it
    for i in range(2):
        assert bool((got[i] - want[i][:, None]).abs().max() <= 64 * U * c.v.double().abs().max())


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("size", [1e5, 1e7, 1e9, 1e12, 1e25])
def test_attention_huge_scores(cuda, kv, size):
    """Where the largest score leads by more than its rounding (and 40: e^-40 < 2^-57), it takes all the weight and all
    of the mass, however large the scores are."""
    c = Cache(cuda, kv, 16, 2, 128, 16, [300, 77, 1], seed=44)
    q = size * cuda.randn(3, 2048, device="cuda")
    k, v = c.host()
    before = c.mass.double().cpu().numpy()
    got = c.attend(q).double().cpu().numpy().reshape(3, 16, 128)
    qq, seen, add = q.double().cpu().numpy().reshape(3, 16, 128), 0, np.zeros_like(before)
    for i in range(3):
        j, p, s = c.places(i)
        for h in range(16):
            kk = k[p, s, h // 8]
            sc = kk @ qq[i, h] * 128 ** -0.5
            ds = 8 * np.sqrt(128) * U * 128 ** -0.5 * (np.abs(kk) @ np.abs(qq[i, h])).max()
            top = sc.argmax()
            if j.size == 1 or sc[top] - np.delete(sc, top).max() > 40 + 2 * ds:
                seen += 1
                assert np.allclose(got[i, h], v[p, s, h // 8][top], rtol=8 * U, atol=8 * U)
                add[p[top], h // 8, s[top]] += 1
            else:
                add[p, h // 8, s] = np.nan   # undecided
    assert seen > 40
    m = c.mass.double().cpu().numpy()
    decided = ~np.isnan(add)
    assert np.isfinite(m).all() and np.all(np.abs(m - before - add)[decided] <= 64 * U * (before + 8)[decided])


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_attention_values_that_are_not_finite_stay_in_their_head(cuda, kv, bad):
    """One infinite or NaN element of K or of V at a visible position: other KV heads, other sequences and, for V, other
    dims keep their bits; masses of the other KV head too."""
    def fresh():
        return Cache(cuda, kv, 16, 2, 128, 16, [300, 77], seed=43)
    q = cuda.randn(2, 2048, device="cuda")
    c = fresh()
    want, mass = c.attend(q).view(2, 2, 8, 128), c.mass.clone()
    _, p, s = c.places(0)
    for pool in ("k", "v"):
        d = fresh()
        getattr(d, pool)[int(p[150]), int(s[150]), 1, 5] = bad
        got = d.attend(q).view(2, 2, 8, 128)
        assert cuda.equal(got[1], want[1]) and cuda.equal(got[0, 0], want[0, 0])
        assert cuda.equal(d.mass[:, 0], mass[:, 0])
        if pool == "v":
            other = cuda.arange(128, device="cuda") != 5
            assert cuda.equal(got[0, 1][:, other], want[0, 1][:, other]) and cuda.equal(d.mass, mass)
            assert not bool(cuda.isfinite(got[0, 1, :, 5]).any())


def test_attention_same_bits_and_no_trace_of_other_calls(cuda):
    """Equal inputs give equal bits, whatever ran on the workspace in between, on another stream too."""
    c = Cache(cuda, "f16", 16, 2, 128, 16, [3000, 5, 1200, 0, 64], seed=11, mass=False)
    q = cuda.randn(5, 2048, device="cuda")
    want = c.attend(q).clone()
    c.attend(cuda.randn(5, 2048, device="cuda"), lens=[7, 2900, 3, 64, 1000])
    assert cuda.equal(c.attend(q), want)
    side = cuda.cuda.Stream()
    side.wait_stream(cuda.cuda.current_stream())
    assert cuda.equal(c.attend(q, stream=side.cuda_stream), want)


def test_attention_graph_replay_with_growing_lengths(cuda):
    c = Cache(cuda, "f16", 16, 2, 128, 16, [500, 40], seed=12, mass=False)
    q, out = cuda.randn(2, 2048, device="cuda"), cuda.empty(2, 2048, device="cuda")
    c.attend(q, out=out)
    g = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(g):
        c.E.paged_attention(c.cfg, c.pool, c.t_dev.data_ptr(), c.l_dev.data_ptr(), 2, q.data_ptr(), out.data_ptr(),
                            c.ws.data_ptr(), c.ws.numel(), stream=cuda.cuda.current_stream().cuda_stream)
    l_dev, t_dev = c.l_dev, c.t_dev
    for lens in ([1, 40], [333, 0], [500, 17]):
        l_dev.copy_(cuda.tensor(lens, dtype=cuda.int32))
        g.replay()
        cuda.cuda.synchronize()
        assert cuda.equal(out, c.attend(q, lens=lens))
    del t_dev


def test_attention_many_sequences(cuda):
    """More sequences than a CTA has threads, empty ones among them."""
    lens = [(37 * i) % 90 if i % 5 else 0 for i in range(600)]
    c = Cache(cuda, "f16", 4, 2, 64, 16, lens, seed=17)
    check_attention(c, cuda.randn(600, 4 * 64, device="cuda"))


@pytest.mark.parametrize("kv,n_head_kv,lens", [("f16", 1, [40000]), ("f32", 2, [30011, 3, 20000]), ("bf16", 1, [9000, 9001])])
def test_attention_long_splits(cuda, kv, n_head_kv, lens):
    """Sequences that all CTAs share: several levels of joins, and masses of positions beyond one CTA's reach."""
    c = Cache(cuda, kv, 8 * n_head_kv, n_head_kv, 128, 64, lens, seed=18)
    check_attention(c, cuda.randn(len(lens), 8 * n_head_kv * 128, device="cuda"))


def test_attention_shared_prefix_pages(cuda):
    """Two sequences whose first pages are the same pages (no mass is kept)."""
    c = Cache(cuda, "f32", 16, 2, 128, 16, [100, 100], seed=13, mass=False)
    c.table[1, :4] = c.table[0, :4]
    check_attention(c, cuda.randn(2, 2048, device="cuda"))


def test_attention_offsets_beyond_32_bits(cuda):
    """Pages 2^31 elements apart: element and byte offsets of the last ones exceed 32 bits."""
    if cuda.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 26 GB")
    from mcpm import engine as E
    stride = 2 ** 31
    big = cuda.empty(6 * stride, dtype=cuda.float16, device="cuda")
    c = Cache(cuda, "f16", 16, 2, 128, 16, [40], seed=14, mass=False, spare=0)
    small = (c.k, c.v)
    views = []
    for i, x in enumerate(small):
        w = cuda.as_strided(big, (3, 16, 2, 128), (stride, 256, 128, 1), i * 3 * stride)
        w.copy_(x)
        views.append(w)
    q = cuda.randn(1, 2048, device="cuda")
    want = c.attend(q).clone()
    c.k, c.v = views
    c.make(1)
    assert cuda.equal(c.attend(q), want)
    assert E.paged_workspace_bytes(c.cfg) > 0


@pytest.mark.parametrize("group,dim", [(8, 128), (3, 64)])
def test_mass_adds_up(cuda, group, dim):
    """The weights that one call adds sum to the query heads of a KV head, and calls accumulate."""
    c = Cache(cuda, "f16", 2 * group, 2, dim, 16, [777, 1, 64], seed=15)
    c.mass.zero_()
    q = cuda.randn(3, 2 * group * dim, device="cuda")
    for k in (1, 2, 3):
        c.attend(q)
        for i in range(3):
            _, p, s = c.places(i)
            got = c.mass.double().cpu().numpy()[p, :, s].sum(0)
            assert np.all(np.abs(got - k * group) <= k * group * 16 * np.sqrt(777) * U)


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_head,n_head_kv,dim,page,split", [(16, 2, 128, 16, False), (12, 4, 64, 7, True), (5, 5, 64, 1, False)])
def test_append(cuda, kv, n_head, n_head_kv, dim, page, split):
    c = Cache(cuda, kv, n_head, n_head_kv, dim, page, [40, 1, 23], seed=page, split=split)
    rng = np.random.default_rng(3)
    seq = np.concatenate([np.full(n, i) for i, n in enumerate(c.lens)]).astype(np.int32)
    slot = np.concatenate([np.arange(n) for n in c.lens]).astype(np.int32)
    order = rng.permutation(seq.size)
    seq, slot = seq[order], slot[order]
    pos = (slot + rng.integers(0, 50, seq.size)).astype(np.int32)
    n, row = seq.size, (n_head + 2 * n_head_kv) * dim
    qkv = cuda.from_numpy(rng.normal(0, 2, (n, row)).astype(np.float32)).cuda()
    rope_host = c.E.rope_table(100, dim)
    d = [c.dev(x) for x in (seq, slot, pos, rope_host, c.table)]
    q_out = cuda.zeros(n, n_head * dim, device="cuda")
    k0, v0, m0 = c.k.clone(), c.v.clone(), c.mass.clone()
    q_ptr = qkv.data_ptr()
    c.E.paged_append(c.cfg, c.pool, d[4].data_ptr(), n, d[1].data_ptr(), q_ptr + 4 * n_head * dim,
                     q_ptr + 4 * (n_head + n_head_kv) * dim, tok_seq=d[0].data_ptr(), tok_pos=d[2].data_ptr(), q=q_ptr,
                     q_out=q_out.data_ptr(), q_stride=row, kv_stride=row, rope=d[3].data_ptr(), rope_len=100)
    cuda.cuda.synchronize()
    x = qkv.double().cpu().numpy().reshape(n, -1, dim)
    cs, sn = (rope_host[pos].astype(np.float64)[..., i][:, None] for i in (0, 1))
    a, b = x[..., 0::2], x[..., 1::2]
    turned, size = np.empty_like(x), np.empty_like(x)
    turned[..., 0::2], turned[..., 1::2] = cs * a - sn * b, sn * a + cs * b
    size[..., 0::2], size[..., 1::2] = np.abs(cs * a) + np.abs(sn * b), np.abs(sn * a) + np.abs(cs * b)
    got_q = q_out.double().cpu().numpy().reshape(n, n_head, dim)
    assert np.all(np.abs(got_q - turned[:, :n_head]) <= 2 * 2.0 ** -24 * size[:, :n_head])   # two roundings
    page_of, at = c.table[seq, slot // page], slot % page
    got_k = c.k.double().cpu().numpy()[page_of, at]
    kt, ks = turned[:, n_head:n_head + n_head_kv], size[:, n_head:n_head + n_head_kv]
    assert np.all(np.abs(got_k - kt) <= HALF_ULP[kv] * np.abs(kt) + 2 * 2.0 ** -23 * ks + 2.0 ** -25)
    want_v = qkv.view(n, -1, dim)[:, n_head + n_head_kv:].to(c.v.dtype)
    p_dev, s_dev = c.dev(page_of).long(), c.dev(at).long()
    assert cuda.equal(c.v[p_dev, s_dev], want_v)
    assert not c.mass[p_dev, :, s_dev].any()
    # nothing else was written
    k0[p_dev, s_dev], v0[p_dev, s_dev] = c.k[p_dev, s_dev], c.v[p_dev, s_dev]
    m0[p_dev, :, s_dev] = 0
    assert cuda.equal(k0, c.k) and cuda.equal(v0, c.v) and cuda.equal(m0, c.mass)


def test_append_matches_the_contiguous_op_bit_for_bit(cuda):
    """The same rotation as mcpm_rope_kv_append, whose cache is one contiguous array."""
    c = Cache(cuda, "f32", 16, 2, 128, 16, [64], seed=2)
    q, k, v = (cuda.randn(n, device="cuda") for n in (2048, 256, 256))
    rope = c.dev(c.E.rope_table(4000))
    for pos in (0, 37, 3999):
        q1, k1 = q.clone(), k.clone()
        kc, vc = cuda.zeros(4000, 256, device="cuda"), cuda.zeros(4000, 256, device="cuda")
        c.E.rope_kv_append(q1.data_ptr(), k1.data_ptr(), v.data_ptr(), kc.data_ptr(), vc.data_ptr(), pos, 4000)
        q2, slot, at = q.clone(), c.dev(np.array([37], np.int32)), c.dev(np.array([pos], np.int32))
        t = c.dev(c.table)
        c.E.paged_append(c.cfg, c.pool, t.data_ptr(), 1, slot.data_ptr(), k.data_ptr(), v.data_ptr(), tok_pos=at.data_ptr(),
                         q=q2.data_ptr(), q_out=q2.data_ptr(), rope=rope.data_ptr(), rope_len=4000)
        cuda.cuda.synchronize()
        p = int(c.table[0, 37 // 16])
        assert cuda.equal(q1, q2)
        assert cuda.equal(c.k[p, 37 % 16].flatten(), kc[pos]) and cuda.equal(c.v[p, 37 % 16].flatten(), vc[pos])


def test_append_padding_and_defaults(cuda):
    """Negative slots, slots beyond the table, absent pages and foreign sequences write nothing; without
    tok_seq, tok_pos, rope and q the rows go in as they are."""
    c = Cache(cuda, "f32", 16, 2, 128, 16, [64, 64, 64, 64, 64], seed=4, mass=False)
    c.table[2, 1] = -1
    k, v = cuda.randn(5, 256, device="cuda"), cuda.randn(5, 256, device="cuda")
    slot = c.dev(np.array([-1, 64, 20, 2 ** 31 - 1, 33], np.int32))
    before, t = (c.k.clone(), c.v.clone()), c.dev(c.table)
    c.E.paged_append(c.cfg, c.pool, t.data_ptr(), 5, slot.data_ptr(), k.data_ptr(), v.data_ptr())
    c.E.paged_append(c.cfg, c.pool, t.data_ptr(), 0, slot.data_ptr(), k.data_ptr(), v.data_ptr())
    seq = c.dev(np.array([-1, 5, 2 ** 31 - 1], np.int32))
    c.E.paged_append(c.cfg, c.pool, t.data_ptr(), 3, c.dev(np.array([1, 2, 3], np.int32)).data_ptr(), k.data_ptr(), v.data_ptr(),
                     tok_seq=seq.data_ptr())
    cuda.cuda.synchronize()
    p = int(c.table[4, 2])
    before[0][p, 1], before[1][p, 1] = k[4].view(2, 128), v[4].view(2, 128)
    assert cuda.equal(before[0], c.k) and cuda.equal(before[1], c.v)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("seqs", [False, True])
def test_append_leaves_the_queries_of_padding_alone(cuda, in_place, seqs):
    """A padding token's row of q_out keeps what it held, with and without tok_pos; a token whose page is absent has its
    query rotated."""
    c = Cache(cuda, "f16", 4, 2, 64, 16, [64] * 6, seed=40)
    c.table[3, 0] = -1
    q, k, v = cuda.randn(6, 256, device="cuda"), cuda.randn(6, 128, device="cuda"), cuda.randn(6, 128, device="cuda")
    slot = np.array([5, -1, 9, 3, -2 ** 31, 64], np.int32)
    seq = np.array([0, 1, 6 if seqs else 2, 3, 4, 5], np.int32)
    q0, pad = q.clone(), np.array([1, 2, 4] if seqs else [1, 4])
    out = q if in_place else cuda.full_like(q, 7.0)
    rope = c.dev(c.E.rope_table(100, 64))
    d = [c.dev(x) for x in (slot, seq, c.table)]
    k1, v1 = c.k.clone(), c.v.clone()
    c.E.paged_append(c.cfg, c.pool, d[2].data_ptr(), 6, d[0].data_ptr(), k.data_ptr(), v.data_ptr(), tok_seq=d[1].data_ptr() if seqs else 0,
                     q=q.data_ptr(), q_out=out.data_ptr(), rope=rope.data_ptr(), rope_len=100)
    cuda.cuda.synchronize()
    real = np.setdiff1d(np.arange(6), pad)
    assert cuda.equal(out[c.dev(pad)], q0[c.dev(pad)] if in_place else cuda.full_like(q0[:pad.size], 7.0))
    cs = c.dev(c.E.rope_table(100, 64)[slot[real]]).double()[:, None]
    a, b = q0[c.dev(real)].double().view(-1, 4, 32, 2).unbind(-1)
    want = cuda.stack([cs[..., 0] * a - cs[..., 1] * b, cs[..., 1] * a + cs[..., 0] * b], -1)
    size = cuda.stack([(cs[..., 0] * a).abs() + (cs[..., 1] * b).abs(), (cs[..., 1] * a).abs() + (cs[..., 0] * b).abs()], -1)
    got = out[c.dev(real)].double().view(-1, 4, 32, 2)
    assert bool(((got - want).abs() <= 2 * 2.0 ** -24 * size).all())   # two roundings
    for i in real:
        if slot[i] < 64 and c.table[i, slot[i] // 16] >= 0:
            p = int(c.table[i, slot[i] // 16])
            k1[p, slot[i] % 16], v1[p, slot[i] % 16] = c.k[p, slot[i] % 16], c.v[p, slot[i] % 16]
            assert cuda.equal(c.v[p, slot[i] % 16], v[i].view(2, 64).half())
    assert cuda.equal(k1, c.k) and cuda.equal(v1, c.v)


# ------------------------------------------------------------------ eviction
def expected_kept(mass, j, n, keep, sink, recent):
    m = mass.astype(np.float64).copy()
    m[np.isnan(m)] = -np.inf
    nan = np.isnan(mass)
    held = (j < sink) | (j >= n - recent)
    order = sorted(range(j.size), key=lambda i: (not held[i], nan[i], -m[i], j[i]))
    return np.sort(j[order[:keep]])


def run_evict(c, dst, keep, sink, recent):
    n = len(c.lens)
    kept = c.torch.full((n, c.n_head_kv, keep), -7, dtype=c.torch.int32, device="cuda")
    new_len = c.torch.full((n,), -7, dtype=c.torch.int32, device="cuda")
    t, d, ln = c.dev(c.table), c.dev(dst), c.dev(np.array(c.lens, np.int32))
    c.E.paged_evict(c.cfg, c.pool, t.data_ptr(), ln.data_ptr(), d.data_ptr(), new_len.data_ptr(), kept.data_ptr(), n, keep,
                    sink, recent, c.ws.data_ptr(), c.ws.numel())
    c.torch.cuda.synchronize()
    return kept.cpu().numpy(), new_len.cpu().numpy()


def check_evict(c, keep, sink, recent):
    n = len(c.lens)
    need = -(-keep // c.page)
    dst = np.full((n, c.cols), -1, np.int32)
    free = list(c.free)
    for i in range(n):
        dst[i, :need] = [free.pop() for _ in range(need)]
    k0, v0, m0 = c.k.clone(), c.v.clone(), c.mass.clone()
    kept, new_len = run_evict(c, dst, keep, sink, recent)
    m = m0.cpu().numpy()
    for i in range(n):
        j, p, s = c.places(i)
        length = min(max(0, c.lens[i]), c.cols * c.page)
        for h in range(c.n_head_kv):
            want = expected_kept(m[p, h, s], j, length, keep, sink, recent)
            assert new_len[i] == want.size
            assert np.array_equal(kept[i, h, :want.size], want), (i, h)
            assert np.all(kept[i, h, want.size:] == -1)
            x = np.arange(want.size)
            a, b = dst[i, x // c.page], x % c.page
            src, at = c.table[i, want // c.page], want % c.page
            da, db, sa, sb = (c.dev(y).long() for y in (a, b, src, at))
            k0[da, db, h], v0[da, db, h], m0[da, h, db] = k0[sa, sb, h], v0[sa, sb, h], m0[sa, h, sb]
    assert cuda_equal_nan(c.torch, k0, c.k) and cuda_equal_nan(c.torch, v0, c.v) and cuda_equal_nan(c.torch, m0, c.mass)
    return kept, new_len


def cuda_equal_nan(torch, a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_head_kv,dim,page,split", [(2, 128, 16, False), (4, 64, 7, True), (1, 128, 1, False)])
def test_evict(cuda, kv, n_head_kv, dim, page, split):
    lens = [0, 1, 60, 99, 100, 101, 500, 1025]
    c = Cache(cuda, kv, 4 * n_head_kv, n_head_kv, dim, page, lens, seed=page, split=split, spare=8 * (100 // page + 1))
    check_evict(c, 100, 4, 30)


@pytest.mark.parametrize("n,keep", [(5000, 4999), (40000, 100), (40000, 39000), (70001, 8192), (150001, 1000)])
def test_evict_long(cuda, n, keep):
    c = Cache(cuda, "f16", 2, 1, 64, 64, [n], seed=n, spare=keep // 64 + 2)
    check_evict(c, keep, 3, 33)


def test_evict_long_among_many(cuda):
    """One CTA per (sequence, head), and more positions than it holds keys of."""
    lens = [40000] + [10] * 74
    c = Cache(cuda, "f16", 2, 1, 64, 64, lens, seed=31, spare=75 * 16)
    check_evict(c, 1000, 3, 33)


def test_evict_equal_masses(cuda):
    """All masses equal, in one CTA and in a cluster: the lowest positions stay."""
    for n in (3000, 70000):
        c = Cache(cuda, "f16", 2, 1, 64, 64, [n], seed=n, spare=20)
        c.mass.fill_(0.0)
        check_evict(c, 1111, 5, 50)


@pytest.mark.parametrize("keep,sink,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (64, 32, 32), (64, 0, 64), (300, 0, 0), (320, 5, 5)])
def test_evict_budgets(cuda, keep, sink, recent):
    c = Cache(cuda, "f32", 16, 2, 128, 16, [300, 200], cols=20, seed=keep, spare=2 * (keep // 16 + 1))
    check_evict(c, keep, sink, recent)


def test_evict_ties_and_special_masses(cuda):
    """Equal masses keep the lowest positions; infinities, negatives, both zeros and NaN have their places."""
    c = Cache(cuda, "f16", 4, 2, 64, 16, [400, 400, 400], seed=1, spare=3 * 8)
    special = np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, -1.0, 1.0, 1e-45, -1e-45, 3.4e38], np.float32)
    m = c.mass.cpu().numpy()
    for i in range(3):
        j, p, s = c.places(i)
        for h in range(2):
            m[p, h, s] = [0.25, special[j % 10], np.where(j % 3 == 0, np.nan, -0.0)][i] if i else 0.25
    c.mass.copy_(cuda.from_numpy(m))
    check_evict(c, 120, 2, 10)


def test_evict_absent_pages(cuda):
    c = Cache(cuda, "f32", 4, 2, 64, 16, [300, 300, 100], seed=3, spare=3 * 7)
    c.table[0, 2], c.table[0, 18], c.table[1, :17] = -1, -1, c.n_pages
    kept, new_len = check_evict(c, 100, 40, 20)
    assert new_len.tolist() == [100, 28, 100]


def test_evict_destination_without_pages_drops_rows(cuda):
    """Rows whose place lies in an absent page are dropped; the rest, kept and new_len are as ever."""
    c = Cache(cuda, "f32", 4, 2, 64, 16, [300], seed=3, spare=8)
    dst = np.full((1, c.cols), -1, np.int32)
    dst[0, :3] = c.free[:3]
    k0 = c.k.clone()
    kept, new_len = run_evict(c, dst, 100, 0, 0)
    assert new_len[0] == 100
    for x in range(48):
        for h in range(2):
            j = kept[0, h, x]
            k0[dst[0, x // 16], x % 16, h] = k0[c.table[0, j // 16], j % 16, h]
    assert cuda.equal(k0, c.k)


def test_attention_after_eviction_sees_the_kept_positions(cuda):
    """Attention over the new pages equals attention over the kept rows alone."""
    c = Cache(cuda, "f32", 16, 2, 128, 16, [250, 90], seed=21, spare=16)
    dst = np.full((2, c.cols), -1, np.int32)
    dst[0, :7], dst[1, :7] = c.free[:7], c.free[7:14]
    _, new_len = run_evict(c, dst, 100, 4, 20)
    assert new_len.tolist() == [100, 90]
    c.table, c.lens = dst, new_len.tolist()
    check_attention(c, cuda.randn(2, 2048, device="cuda"))
