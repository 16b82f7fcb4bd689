"""Variants and faults of the paged-cache kernels that the general tests do not reach: every group size, errors next to
those of an fp32 form, every tile of long sequences, many pairs, calls in graphs and on other streams."""
import numpy as np
import pytest

from test_gpu_paged import U, Cache, check_attention, check_evict, expected_kept

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("mass", [True, False])
@pytest.mark.parametrize("group", [2, 4, 5, 6, 7, 9, 10, 11, 12, 13, 14, 15, 16])
def test_group_sizes(cuda, kv, mass, group):
    for n_head_kv, dim in ((2, 128), (3, 64)):
        c = Cache(cuda, kv, group * n_head_kv, n_head_kv, dim, 16, [1, 0, 17, 130, 777, 2049], seed=group, mass=mass)
        check_attention(c, 1.5 * cuda.randn(6, group * n_head_kv * dim, device="cuda"))


def fp32_form(c, q, scale):
    """Attention in elementary fp32 torch operations on the cache's values, a sequence and a KV head at a time."""
    torch, g = c.torch, c.n_head // c.n_head_kv
    out = torch.zeros(len(c.lens), c.n_head, c.dim, device="cuda")
    for i in range(len(c.lens)):
        _, p, s = c.places(i)
        if p.size == 0:
            continue
        p, s = c.dev(p).long(), c.dev(s).long()
        for h in range(c.n_head_kv):
            score = scale * (q[i].view(c.n_head, c.dim)[h * g:(h + 1) * g] @ c.k[p, s, h].float().T)
            e = (score - score.amax(1, keepdim=True)).exp()
            out[i, h * g:(h + 1) * g] = (e / e.sum(1, keepdim=True)) @ c.v[p, s, h].float()
    return out.view(len(c.lens), -1)


def exact_form(c, q, scale):
    g, n = c.n_head // c.n_head_kv, len(c.lens)
    out = c.torch.zeros(n, c.n_head, c.dim, dtype=c.torch.float64, device="cuda")
    for i in range(n):
        _, p, s = c.places(i)
        if p.size == 0:
            continue
        p, s = c.dev(p).long(), c.dev(s).long()
        for h in range(c.n_head_kv):
            score = scale * (q[i].double().view(c.n_head, c.dim)[h * g:(h + 1) * g] @ c.k[p, s, h].double().T)
            out[i, h * g:(h + 1) * g] = c.torch.softmax(score, 1) @ c.v[p, s, h].double()
    return out.view(n, -1)


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_head,n_head_kv,dim", [(16, 2, 128), (16, 1, 128), (12, 4, 64), (3, 1, 128), (30, 2, 64)])
@pytest.mark.parametrize("lens", [[15, 100, 333], [1500, 2048], [40000]])
def test_errors_are_those_of_an_fp32_form(cuda, kv, n_head, n_head_kv, dim, lens):
    """Root mean square error against 64 bits next to an fp32 form's on the same inputs: the kernel rounds scores, weights
    and sums as that does, in another order and with accumulators that truncate (2^-23 for 2^-24): at most twice the
    form's, and three times for an fp32 cache, which is itself split in two parts of 11 bits without the product of the
    lower ones.  In fp32 arithmetic with a part left out, on inputs like these, the error is 180 to 840 times the form's
    for the second part of q or of the weights (fp16, tf32), 4 to 10 times for the third bf16 part of q, and 3 to 4 times
    for the third one of the weights."""
    c = Cache(cuda, kv, n_head, n_head_kv, dim, 16, lens, seed=len(lens), mass=False)
    cuda.manual_seed(7)
    q = 1.5 * cuda.randn(len(lens), n_head * dim, device="cuda")
    scale = dim ** -0.5
    was = cuda.backends.cuda.matmul.allow_tf32
    cuda.backends.cuda.matmul.allow_tf32 = False
    plain, want = fp32_form(c, q, scale), exact_form(c, q, scale)
    cuda.backends.cuda.matmul.allow_tf32 = was
    got = c.attend(q)

    def rms(x):
        return float((x.double() - want).square().mean().sqrt())

    assert rms(got) <= (3 if kv == "f32" else 2) * rms(plain), (rms(got), rms(plain))


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("group", [8, 3, 16])
@pytest.mark.parametrize("case", ["one long", "two long", "very long", "ragged", "short"])
def test_every_tile_counts_once(cuda, kv, group, case):
    """Equal scores, and V a one in the dim that a position's tile of 16 names: an output is the share of its dim's
    positions, sums of ones that fp32 holds exactly and one quotient (three roundings).  A tile that is missing, or there
    twice, is 16 positions of at most 1100.  Masses are group / length, a sum of `group` rounded quotients."""
    rng = np.random.default_rng(3)
    lens = {"one long": [40000], "two long": [30011, 3, 20000], "very long": [140001], "ragged": list(rng.integers(300, 4097, 64)),
            "short": list(rng.integers(1, 900, 200))}[case]
    lens = [int(n) for n in lens]
    c = Cache(cuda, kv, group, 1, 128, 64, lens, seed=11, pool_fill=1.0)
    c.mass.zero_()
    want = np.zeros((len(lens), 128))
    for i, n in enumerate(lens):
        j, p, s = c.places(i)
        mark = cuda.zeros(n, 1, 128, dtype=c.v.dtype, device="cuda")
        mark[cuda.arange(n, device="cuda"), 0, c.dev(j // 16 % 128).long()] = 1
        c.v[c.dev(p).long(), c.dev(s).long()] = mark
        want[i] = np.bincount(j // 16 % 128, minlength=128) / n
    got = c.attend(cuda.zeros(len(lens), group * 128, device="cuda")).double().cpu().numpy().reshape(len(lens), group, 128)
    assert np.all(np.abs(got - want[:, None]) <= 4 * U * want[:, None])
    m = c.mass.double().cpu().numpy()
    for i, n in enumerate(lens):
        _, p, s = c.places(i)
        assert np.all(np.abs(m[p, 0, s] - group / n) <= (group + 3) * U * group / n)
        m[p, 0, s] = 0
    assert not m.any()


@pytest.mark.parametrize("n_head_kv,dim,lens,keep", [
    (2, 64, [int(n) for n in np.random.default_rng(1).integers(1, 2700, 100)], 700),   # 200 pairs
    (1, 128, [0] * 3 + [40000] + [33 * i % 400 for i in range(156)], 300),             # more keys than a CTA holds
    (149, 64, [50, 321], 64)])
def test_evict_more_pairs_than_sms(cuda, n_head_kv, dim, lens, keep):
    assert len(lens) * n_head_kv > cuda.cuda.get_device_properties(0).multi_processor_count
    c = Cache(cuda, "f16", n_head_kv, n_head_kv, dim, 16, lens, seed=51, spare=len(lens) * -(-keep // 16))
    check_evict(c, keep, 3, 20)


def test_evict_many_equal_and_special_masses(cuda):
    """More pairs than SMs whose masses are ties, NaN, infinities and zeros, with absent pages."""
    c = Cache(cuda, "bf16", 2, 2, 64, 16, [400] * 80, seed=52, spare=80 * 8)
    m = c.mass.cpu().numpy()
    special = np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, -1.0, 1.0, 1e-45, 0.5, 0.5], np.float32)
    for i in range(80):
        j, p, s = c.places(i)
        m[p, 0, s], m[p, 1, s] = special[(j * (i + 1)) % 10], 0.25 if i % 2 else special[j % 3]
        if i % 5 == 0:
            c.table[i, i % 25] = -1
    c.mass.copy_(cuda.from_numpy(m))
    check_evict(c, 120, 2, 10)


def test_append_attention_and_eviction_in_a_graph(cuda):
    """One step captured once and replayed with other lengths, slots, tables and rows: the bits of eager calls."""
    def fresh():
        c = Cache(cuda, "f16", 16, 2, 128, 16, [200, 75, 31], seed=61, spare=24)
        return c, [c.dev(x) for x in (c.table, np.array(c.lens, np.int32), np.zeros(3, np.int32), np.full((3, c.cols), -1, np.int32))]

    def buffers():
        f = dict(device="cuda")
        return (cuda.zeros(3, 2560, **f), cuda.zeros(3, 2048, **f), cuda.zeros(3, 2048, **f), cuda.zeros(3, dtype=cuda.int32, **f),
                cuda.zeros(3, 2, 64, dtype=cuda.int32, **f))

    def step(c, dev, b, stream):
        table, length, slot, dst = dev
        qkv, q, out, new_len, kept = b
        at = qkv.data_ptr()
        c.E.paged_append(c.cfg, c.pool, table.data_ptr(), 3, slot.data_ptr(), at + 4 * 2048, at + 4 * 2304, q=at, q_out=q.data_ptr(), q_stride=2560,
                         kv_stride=2560, rope=rope.data_ptr(), rope_len=300, stream=stream)
        c.E.paged_attention(c.cfg, c.pool, table.data_ptr(), length.data_ptr(), 3, q.data_ptr(), out.data_ptr(), c.ws.data_ptr(), c.ws.numel(), stream=stream)
        c.E.paged_evict(c.cfg, c.pool, table.data_ptr(), length.data_ptr(), dst.data_ptr(), new_len.data_ptr(), kept.data_ptr(), 3, 64, 4, 16,
                        c.ws.data_ptr(), c.ws.numel(), stream=stream)

    (a, da), (b, db) = fresh(), fresh()
    rope = a.dev(a.E.rope_table(300))
    ba, bb = buffers(), buffers()
    step(a, da, ba, cuda.cuda.current_stream().cuda_stream)   # kernels are loaded; then the same cache on both sides
    cuda.cuda.synchronize()
    a.k.copy_(b.k), a.v.copy_(b.v), a.mass.copy_(b.mass)
    graph = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(graph):
        step(a, da, ba, cuda.cuda.current_stream().cuda_stream)
    dst = np.full((3, a.cols), -1, np.int32)
    for t in range(3):
        dst[:, :4] = np.array(a.free[12 * (t % 2):12 * (t % 2) + 12]).reshape(3, 4)
        lens = np.array([[200, 75, 31], [57, 0, 20], [130, 74, 5]][t], np.int32)
        rows = cuda.randn(3, 2560, device="cuda")
        for dev, buf in ((da, ba), (db, bb)):
            dev[1].copy_(cuda.from_numpy(lens))
            dev[2].copy_(cuda.from_numpy(lens - 1))   # -1: padding
            dev[3].copy_(cuda.from_numpy(dst))
            buf[0].copy_(rows)
        graph.replay()
        cuda.cuda.synchronize()
        step(b, db, bb, 0)
        cuda.cuda.synchronize()
        for x, y in zip(ba, bb):
            assert cuda.equal(x, y)
        assert cuda.equal(a.k, b.k) and cuda.equal(a.v, b.v) and cuda.equal(a.mass, b.mass)
        assert ba[3].tolist() == [min(64, n) for n in lens]


def test_eviction_on_a_side_stream(cuda):
    """Behind work of its own stream that writes the lengths and the masses, beside other work of the default one."""
    c = Cache(cuda, "f32", 4, 2, 64, 16, [3000, 500], seed=62, spare=20)
    m0, k0 = c.mass.clone(), c.k.clone()
    side = cuda.cuda.Stream()
    t, ln = c.dev(c.table), cuda.zeros(2, dtype=cuda.int32, device="cuda")
    dst = np.full((2, c.cols), -1, np.int32)
    dst[0, :8], dst[1, :8] = c.free[:8], c.free[8:16]
    d, new_len, kept = c.dev(dst), cuda.zeros(2, dtype=cuda.int32, device="cuda"), cuda.zeros(2, 2, 120, dtype=cuda.int32, device="cuda")
    lens, scale = c.dev(np.array(c.lens, np.int32)), cuda.randn(1 << 22, device="cuda")
    cuda.cuda.synchronize()
    with cuda.cuda.stream(side):
        for _ in range(20):
            scale.mul_(1.0)
        ln.copy_(lens)
        c.mass.mul_(-1.0)
        c.E.paged_evict(c.cfg, c.pool, t.data_ptr(), ln.data_ptr(), d.data_ptr(), new_len.data_ptr(), kept.data_ptr(), 2, 120, 4, 16,
                        c.ws.data_ptr(), c.ws.numel(), stream=side.cuda_stream)
        got = kept.clone()
    side.synchronize()
    assert new_len.tolist() == [120, 120]
    m = -m0.cpu().numpy()
    for i in range(2):
        j, p, s = c.places(i)
        for h in range(2):
            want = expected_kept(m[p, h, s], j, c.lens[i], 120, 4, 16)
            assert np.array_equal(got[i, h].cpu().numpy(), want)
            x = np.arange(120)
            a, b = c.dev(dst[i, x // 16]).long(), c.dev(x % 16).long()
            src, at = c.dev(c.table[i, want // 16]).long(), c.dev(want % 16).long()
            assert cuda.equal(c.k[a, b, h], k0[src, at, h])
