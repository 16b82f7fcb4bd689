"""mcpm_logits_process: refusals on the CPU; on the GPU the values against a plain 64-bit implementation
(each of at most six fp32 operations errs by 2^-24 of its result, and no intermediate exceeds the sum of the
magnitudes below) and the greedy token against the row that came out."""
import numpy as np
import pytest

NEG_INF = -np.inf


def plain(x, hist, pen, bias_token, bias, allow):
    x = x.astype(np.float64)
    size = np.abs(x)
    if hist is not None:
        hist = hist[(hist >= 0) & (hist < x.size)]
        c = np.bincount(hist, minlength=x.size).astype(np.float64)
        rep, freq, pres = (float(p) for p in pen)
        y = np.where(x > 0, x / rep, x * rep) - (freq * c + pres)
        with np.errstate(invalid="ignore"):
            size = np.where(c > 0, np.maximum(size, size * max(rep, 1 / rep)) + abs(freq) * c + abs(pres), size)
        x = np.where(c > 0, y, x)
    if bias_token is not None:
        for t, b in {int(t): float(b) for t, b in zip(bias_token, bias)}.items():
            if 0 <= t < x.size:
                x[t] += b
                size[t] += abs(b)
    x = np.where(np.abs(x) > np.finfo(np.float32).max, np.copysign(np.inf, x), x)   # what an fp32 result holds
    if allow is not None:
        bits = np.unpackbits(allow.view(np.uint8), bitorder="little")[:x.size]
        x[bits == 0] = NEG_INF
    return x, 6 * 2.0 ** -24 * size


class Rows:
    def __init__(self, torch, n, v, hist=0, bias=0, mask=False, seed=0, pad=0):
        rng = np.random.default_rng(seed)
        self.torch, self.n, self.v = torch, n, v
        self.x = rng.normal(0, 3, (n, v + pad)).astype(np.float32)
        self.hist = (v * rng.random((n, max(1, hist))) ** 3).astype(np.int32) if hist else None
        self.hist_len = np.array([hist - (i * hist) // n for i in range(n)], np.int32)
        self.pen = np.stack([1 + rng.random(n), rng.normal(0, 0.5, n), rng.normal(0, 0.5, n)], 1).astype(np.float32)
        self.bias_token = rng.integers(0, v, (n, bias)).astype(np.int32) if bias else None
        self.bias = rng.normal(0, 5, (n, max(1, bias))).astype(np.float32)
        self.bias_len = np.array([bias - i % 2 for i in range(n)], np.int32)
        self.allow = rng.integers(0, 2 ** 32, (n, (v + 31) // 32), dtype=np.uint32) if mask else None

    def run(self, in_place=False, stream=0, **change):
        from mcpm import engine as E
        torch = self.torch
        d = {k: torch.from_numpy(np.ascontiguousarray(a.view(np.int32) if a.dtype == np.uint32 else a)).cuda()
             for k, a in vars(self).items() if isinstance(a, np.ndarray)}
        out = d["x"] if in_place else torch.full_like(d["x"], 9.0)
        token = torch.full((self.n,), -9, dtype=torch.int32, device="cuda")
        more = {}
        if self.hist is not None:
            more.update(hist=d["hist"].data_ptr(), hist_stride=self.hist.shape[1], hist_len=d["hist_len"].data_ptr(), penalties=d["pen"].data_ptr())
        if self.bias_token is not None:
            more.update(bias_token=d["bias_token"].data_ptr(), bias=d["bias"].data_ptr(), bias_stride=self.bias_token.shape[1],
                        bias_len=d["bias_len"].data_ptr())
        if self.allow is not None:
            more.update(allow=d["allow"].data_ptr())
        more.update(change)
        torch.cuda.synchronize()
        E.logits_process(d["x"].data_ptr(), out.data_ptr(), self.n, self.v, argmax=token.data_ptr(), logits_stride=self.x.shape[1],
                         out_stride=self.x.shape[1], stream=stream, **more)
        torch.cuda.synchronize()
        return out.cpu().numpy(), token.cpu().numpy()

    def check(self, in_place=False, stream=0):
        got, token = self.run(in_place, stream)
        for i in range(self.n):
            nh, nb = min(max(self.hist_len[i], 0), 1 << 20), max(0, self.bias_len[i])
            want, tol = plain(self.x[i, :self.v], None if self.hist is None else self.hist[i, :nh], self.pen[i],
                              None if self.bias_token is None else self.bias_token[i, :nb], self.bias[i, :nb],
                              None if self.allow is None else self.allow[i])
            y = got[i, :self.v].astype(np.float64)
            fin = np.isfinite(want)
            assert np.array_equal(np.isnan(y), np.isnan(want)) and np.array_equal(y[~fin & ~np.isnan(want)], want[~fin & ~np.isnan(want)])
            assert np.all(np.abs(y[fin] - want[fin]) <= tol[fin]), np.max(np.abs(y[fin] - want[fin]) - tol[fin])
            best = np.where(np.isnan(y), NEG_INF, y)
            assert token[i] == (best.argmax() if best.max() > NEG_INF else -1)
            assert np.array_equal(got[i, self.v:], (self.x if in_place else np.full_like(self.x, 9.0))[i, self.v:])
        return got, token


@pytest.mark.gpu
@pytest.mark.parametrize("n,v", [(1, 1), (1, 31), (2, 33), (3, 4097), (2, 130560), (5, 32003), (1, 300001)])
@pytest.mark.parametrize("hist,bias,mask", [(0, 0, False), (50, 0, False), (0, 7, False), (0, 0, True), (700, 64, True)])
def test_logits(cuda, n, v, hist, bias, mask):
    Rows(cuda, n, v, hist, bias, mask, seed=v + hist).check()


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [1, 4, 61])
def test_logits_strided_and_in_place(cuda, pad):
    r = Rows(cuda, 4, 5003, 100, 9, True, seed=pad, pad=pad)
    a, ta = r.check()
    b, tb = r.check(in_place=True)
    assert np.array_equal(a[:, :5003], b[:, :5003]) and np.array_equal(ta, tb)


@pytest.mark.gpu
def test_logits_counts_and_history_bounds(cuda):
    """Foreign ids are ignored, lengths clamped, and a long history of one token is counted in full."""
    r = Rows(cuda, 5, 1000, 4096, seed=1)
    r.hist[0, :] = 7
    r.hist[1, ::2] = -1
    r.hist[1, 1::2] = 1000
    r.hist[2, :5] = [2 ** 31 - 1, -2 ** 31, 999, 0, 999]
    r.hist_len[:] = [4096, 4096, 5, 0, -3]
    r.check()
    full, _ = r.run(hist_len=0)
    r.hist_len[:] = 4096
    assert np.array_equal(full, r.check()[0])
    r.hist_len[:] = 2 ** 31 - 1
    assert np.array_equal(full, r.run()[0])


@pytest.mark.gpu
@pytest.mark.parametrize("n,v", [(1, 600001), (9, 300007), (9, 524288)])
def test_logits_large_vocabularies(cuda, n, v):
    """Shares of a CTA beyond one slice."""
    Rows(cuda, n, v, 900, 50, True, seed=v).check()


@pytest.mark.gpu
@pytest.mark.parametrize("n,hist", [(1, 20000), (9, 20000), (2, 9001), (3, 100000)])
def test_logits_long_histories(cuda, n, hist):
    """More entries than one round takes, and more distinct tokens than a slice's list holds."""
    r = Rows(cuda, n, 130560, hist, 300, True, seed=hist)
    r.hist[:] = np.random.default_rng(7).integers(0, 130560, r.hist.shape)
    r.check()


@pytest.mark.gpu
def test_logits_duplicate_and_foreign_biases(cuda):
    r = Rows(cuda, 2, 500, 0, 4094, seed=2)   # most tokens are listed about eight times: the last entry counts
    r.bias_token[0, ::3] = -1
    r.bias_token[1, ::3] = 500
    r.check()


@pytest.mark.gpu
def test_logits_special_values(cuda):
    r = Rows(cuda, 4, 1000, 200, 5, True, seed=3)
    r.x[:, ::7] = np.nan
    r.x[:, 1::7] = np.inf
    r.x[:, 2::7] = -np.inf
    r.x[2] = np.nan
    r.x[3, :] = np.finfo(np.float32).min
    r.check()


@pytest.mark.gpu
def test_logits_ties_and_dead_ends(cuda):
    r = Rows(cuda, 4, 70001, 0, 0, True, seed=4)
    r.x[:] = 1.5
    r.allow[:] = 0
    r.allow[1, -1] = np.uint32(1) << 16       # the last token alone: 70000 = 32 * 2187 + 16
    r.allow[2, 1000] = r.allow[2, 2000] = 12  # equal logits: the lowest of 32002, 32003, 64002, 64003
    r.allow[3, 0] = 0x80000000
    _, token = r.check()
    assert token.tolist() == [-1, 70000, 32002, 31]


@pytest.mark.gpu
@pytest.mark.parametrize("n,v", [(1, 32768), (8, 5001), (9, 5001), (9, 32768), (20, 130560), (64, 8192)])
@pytest.mark.parametrize("hist,bias", [(0, 0), (60, 0), (0, 9), (700, 40)])
@pytest.mark.parametrize("mask", [False, True])
def test_logits_variants(cuda, n, v, hist, bias, mask):
    """Rows of sixteen and of eight CTAs, aligned and odd ones, with and without lists and masks."""
    Rows(cuda, n, v, hist, bias, mask, seed=n + v + hist).check()


@pytest.mark.gpu
@pytest.mark.parametrize("v", [5001, 130560])
def test_logits_do_not_depend_on_the_rows_beside_them(cuda, v):
    """A row alone, among few and among many rows: the same bits, whatever the number of CTAs that share it."""
    r = Rows(cuda, 30, v, 300, 20, True, seed=v)
    all_rows, tokens = r.run()
    for n in (1, 8, 9):
        few = Rows(cuda, n, v, 300, 20, True, seed=v)
        for k in ("x", "hist", "hist_len", "pen", "bias_token", "bias", "bias_len", "allow"):
            setattr(few, k, getattr(r, k)[:n])
        got, token = few.run()
        assert np.array_equal(got, all_rows[:n]) and np.array_equal(token, tokens[:n])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [2, 12])
def test_logits_without_the_greedy_token(cuda, n):
    """The same rows where no greedy token is asked for, whose cluster has nothing to exchange."""
    from mcpm import engine as E
    r = Rows(cuda, n, 9001, 200, 5, True, seed=n)
    want, _ = r.run()
    d = {k: cuda.from_numpy(getattr(r, k).view(np.int32) if k == "allow" else getattr(r, k)).cuda()
         for k in ("x", "hist", "hist_len", "pen", "bias_token", "bias", "bias_len", "allow")}
    out = cuda.zeros(n, 9001, device="cuda")
    E.logits_process(d["x"].data_ptr(), out.data_ptr(), n, 9001, hist=d["hist"].data_ptr(), hist_stride=200, hist_len=d["hist_len"].data_ptr(),
                     penalties=d["pen"].data_ptr(), bias_token=d["bias_token"].data_ptr(), bias=d["bias"].data_ptr(), bias_stride=5,
                     bias_len=d["bias_len"].data_ptr(), allow=d["allow"].data_ptr())
    cuda.cuda.synchronize()
    assert np.array_equal(out.cpu().numpy(), want)


@pytest.mark.gpu
def test_logits_on_a_side_stream_and_in_a_graph(cuda):
    from mcpm import engine as E
    r = Rows(cuda, 3, 9001, 40, 3, True, seed=5)
    want = r.check()
    side = cuda.cuda.Stream()
    got = r.check(stream=side.cuda_stream)
    assert np.array_equal(want[0], got[0]) and np.array_equal(want[1], got[1])
    x, out, tok = cuda.randn(3, 9001, device="cuda"), cuda.zeros(3, 9001, device="cuda"), cuda.zeros(3, dtype=cuda.int32, device="cuda")
    g = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(g):
        E.logits_process(x.data_ptr(), out.data_ptr(), 3, 9001, argmax=tok.data_ptr(), stream=cuda.cuda.current_stream().cuda_stream)
    x.normal_()
    g.replay()
    cuda.cuda.synchronize()
    assert cuda.equal(out, x) and cuda.equal(tok.long(), x.argmax(1))


@pytest.mark.gpu
def test_masked_logits_feed_the_sampler(cuda):
    """A grammar that leaves one token makes the top-p sampler draw it, whatever the draw."""
    from mcpm import engine as E
    r = Rows(cuda, 1, 2000, 0, 0, True, seed=6)
    r.allow[:] = 0
    r.allow[0, 40] = 1 << 9
    got, token = r.check()
    x, out = cuda.from_numpy(got[0]).cuda(), cuda.zeros(2, dtype=cuda.int32, device="cuda")
    for draw in (0.0, 0.5, 0.999):
        E.sample_top_p(x.data_ptr(), 2000, 0.8, 0.9, draw, out.data_ptr())
        assert out[0].item() == token[0] == 40 * 32 + 9


OK_PTR = 256   # never dereferenced: every call below is refused before it reaches the device


@pytest.mark.parametrize("change", [
    dict(n_seq=0), dict(n_seq=-1), dict(n_vocab=0), dict(logits=None), dict(out=None), dict(logits_stride=99),
    dict(out_stride=99), dict(out=OK_PTR, logits=OK_PTR, out_stride=128), dict(hist=OK_PTR, hist_max=5),
    dict(hist=OK_PTR, penalties=OK_PTR, hist_max=-1), dict(hist=OK_PTR, penalties=OK_PTR, hist_max=1 << 20),
    dict(hist=OK_PTR, penalties=OK_PTR, hist_max=9, hist_stride=8), dict(bias_token=OK_PTR, bias_max=3),
    dict(bias_token=OK_PTR, bias=OK_PTR, bias_max=4095), dict(bias_token=OK_PTR, bias=OK_PTR, bias_max=5, bias_stride=4),
    dict(allow=OK_PTR, allow_stride=3), dict(n_vocab=(1 << 30) + 1)])
def test_logits_refusals(change):
    from mcpm import engine as E
    lib = E.load_library()
    p = E.mcpm_logits_params(n_seq=2, n_vocab=100, logits=OK_PTR, out=2 * OK_PTR)
    for k, v in change.items():
        setattr(p, k, v)
    assert lib.mcpm_logits_process(p, None) == E.BAD_ARG
    assert lib.mcpm_logits_process(None, None) == E.BAD_ARG
