"""Decoding over the paged cache: the appended rows against the engine's cache, the logits against the reference
build's goldens under the gate of test_gpu_parity_model.py, evictions, and the logits operator at the end.
"""
import json
import os

import numpy as np
import pytest

from conftest import GOLDEN

PARITY_DSCALE = 0.04


def test_embedding_dequantisation(oracle):
    """Q4_K rows as the restatement reads them: one product and one fma-free difference per value (2^-22 of the
    larger term covers their roundings)."""
    torch = pytest.importorskip("torch")  # noqa: F841  (mcpm.paged imports it)
    from conftest import rand_tensor_bytes
    from mcpm import paged
    raw = rand_tensor_bytes(12, 4, 2048, 3).reshape(-1, 144)
    got = paged.dequantize_q4_k(raw).astype(np.float64)
    # from the format: x = d * scale * q - dmin * min
    for b in range(raw.shape[0]):
        d, dmin = raw[b, :4].copy().view(np.float16).astype(np.float64)
        for i in range(256):
            j = i // 32
            s = raw[b, 4:16].astype(int)
            sc, mn = (s[j] & 63, s[j + 4] & 63) if j < 4 else ((s[j + 4] & 15) | (s[j - 4] >> 6) << 4, (s[j + 4] >> 4) | (s[j] >> 6) << 4)
            byte = int(raw[b, 16 + i // 64 * 32 + i % 32])
            q = byte >> 4 if i % 64 >= 32 else byte & 15
            want = d * sc * q - dmin * mn
            assert abs(got[b, i] - want) <= 2.0 ** -22 * (abs(d * sc * q) + abs(dmin * mn))


@pytest.fixture(scope="module")
def parity():
    g = np.load(os.path.join(GOLDEN, "reference_decode_wc.npz"))
    v = json.load(open(os.path.join(GOLDEN, "reference_variability_wc.json")))
    from mcpm import synth
    return g, v, synth.ensure_model("q4_k_m", 0, dscale=PARITY_DSCALE)


@pytest.mark.gpu
def test_paged_decode_against_the_reference(cuda, parity):
    """All 192 positions, teacher-forced: argmax at the positions that the reference decides, logits within its
    own spread; the first layer's K and V rows are the engine's, bit for bit."""
    from mcpm import engine as E, paged
    g, v, path = parity
    toks, prompt = g["tokens"], g["prompt"]
    n = len(toks)
    inputs = list(prompt) + list(toks[len(prompt) - 1:n - 1])
    d = paged.PagedDecoder(path, n_pages=20, max_positions=256)
    s = d.open()
    am, top = [], []
    for p in range(n):
        am.append(d.step({s: int(inputs[p])})[s])
        top.append(d.logits[0].cpu().numpy()[g["top_idx"][p]])
    am, top, dec = np.array(am), np.array(top), np.array(v["decidable"])
    assert np.array_equal(am[dec], toks[dec])
    assert np.abs(top - g["top_val"]).mean() <= 1.25 * max(v["mean_abs_top32_4_vs_1"])
    eng = E.MiniCPM5Engine(device=0, max_seq=64)
    assert eng.load_model(path)
    for p in range(40):
        eng.forward_greedy(int(inputs[p]), p)
        k, val = eng.read_kv(0, p)
        page, slot = d.table[s, p // 16], p % 16
        assert np.array_equal(d.k[0, page, slot].cpu().numpy().ravel(), k)
        assert np.array_equal(d.v[0, page, slot].cpu().numpy().ravel(), val)
    eng.close()


@pytest.mark.gpu
def test_sequences_of_unlike_lengths_share_the_pool(cuda, parity):
    """Two sequences, opened at different times and stepped together, append what each appends alone."""
    from mcpm import paged, synth
    _, _, path = parity
    ids = [synth.prompt_ids(24, seed=s) for s in (1, 2)]
    alone = []
    for i in (0, 1):
        d = paged.PagedDecoder(path, n_pages=4, max_positions=64)
        s = d.open()
        for t in ids[i][:20 - 4 * i]:
            d.step({s: int(t)})
        alone.append(_rows(d, s))
        d.close(s)
        assert sorted(d.free) == list(range(4))
    d = paged.PagedDecoder(path, n_pages=5, max_positions=64, max_seqs=2)
    a = d.open()
    for t in ids[0][:4]:
        d.step({a: int(t)})
    b = d.open()
    for i in range(16):
        d.step({b: int(ids[1][i]), a: int(ids[0][4 + i])})
    for s, (k, v) in ((a, alone[0]), (b, alone[1])):
        got = _rows(d, s)
        assert np.array_equal(got[0], k) and np.array_equal(got[1], v)   # layer 0: before any attention


def _rows(d, s):
    n = int(d.length[s])
    page, slot = d.table[s, np.arange(n) // d.page_size].astype(np.int64), np.arange(n) % d.page_size
    return d.k[0].cpu().numpy()[page, slot], d.v[0].cpu().numpy()[page, slot]


@pytest.mark.gpu
def test_bounded_cache(cuda, parity):
    """A conversation longer than its cache: evictions keep the sinks and the recent positions in every layer,
    pages come back, masses of kept positions survive, and positions keep counting."""
    from mcpm import paged, synth
    _, _, path = parity
    d = paged.PagedDecoder(path, n_pages=8, max_positions=64, keep=32, slack=16, sink=2, recent=8)
    s = d.open()
    ids = synth.prompt_ids(120, seed=9)
    seen_k = []
    for p, t in enumerate(ids):
        if d.length[s] == 48:
            before = _rows(d, s)[0]
        full = d.length[s] == 48
        token = d.step({s: int(t)})[s]
        assert 0 <= token < d.n_vocab and bool(cuda.isfinite(d.logits).all())
        if full:
            after = _rows(d, s)[0]
            assert d.length[s] == 33
            for h in range(2):
                assert np.array_equal(after[:2, h], before[:2, h]) and np.array_equal(after[24:32, h], before[40:48, h])
            seen_k.append(after[32])
        assert int(d.position[s]) == p + 1 and d.length[s] <= 48
        assert len(d.free) == 8 - -(-int(d.length[s]) // 16)
    assert len(seen_k) == 5
    # each step's weights sum to 8 query heads per KV head, spread over what is visible
    m = d.mass[:, d.table[s, 0]].cpu().numpy()
    assert np.isfinite(m).all() and (m >= 0).all() and m[:, :, 0].max() > 1


@pytest.mark.gpu
def test_penalties_biases_and_grammar_reach_the_token(cuda, parity):
    from mcpm import paged, synth
    _, _, path = parity
    d = paged.PagedDecoder(path, n_pages=8, max_positions=64)
    ids = [int(t) for t in synth.prompt_ids(5, seed=3)]

    def run(**k):
        s = d.open()
        for t in ids[:-1]:
            d.step({s: t})
        token = d.step({s: ids[-1]}, **k)[s]
        lg = d.logits[0].cpu().numpy().copy()
        d.close(s)
        return token, lg

    plain, lg = run()
    assert plain == lg.argmax()
    assert run(bias={plain: -1e4})[0] == np.argsort(-lg)[1]
    assert run(bias={77: 1e4})[0] == 77
    allow = np.zeros(d.n_vocab, bool)
    allow[[5, 130559]] = True
    assert run(allow=allow)[0] == (5 if lg[5] >= lg[130559] else 130559)
    assert run(allow=np.zeros(d.n_vocab, bool))[0] == -1
    pen = lg.astype(np.float64)
    for t in set(ids):
        pen[t] -= 1e3 * ids.count(t)
    assert run(frequency=1e3)[0] == pen.argmax()


@pytest.mark.gpu
def test_paged_decoder_refusals(cuda, parity):
    from mcpm import engine as E, paged
    _, _, path = parity
    with pytest.raises(ValueError):
        paged.PagedDecoder(path, n_pages=4, keep=8, sink=4, recent=8)
    d = paged.PagedDecoder(path, n_pages=1, max_positions=32, max_seqs=1)
    with pytest.raises(E.MCPMError) as e:
        d.step({0: 1})
    assert e.value.status == E.BAD_ARG
    s = d.open()
    with pytest.raises(E.MCPMError):
        d.open()
    with pytest.raises(E.MCPMError) as e:
        d.step({s: d.n_vocab})
    assert e.value.status == E.BAD_TOKEN
    for _ in range(16):
        d.step({s: 1})
    with pytest.raises(E.MCPMError) as e:   # the only page is full
        d.step({s: 1})
    assert e.value.status == E.OOM


@pytest.mark.gpu
def test_a_refused_step_can_be_repeated(cuda, parity):
    """Two sequences at the end of their first page, a bad token and a pool without room: nothing is taken or lost,
    the step made good writes what an undisturbed one writes, and every page comes back."""
    from mcpm import engine as E, paged, synth
    _, _, path = parity
    ids = [[int(t) for t in synth.prompt_ids(17, seed=s)] for s in (4, 5)]

    def start(n_pages):
        d = paged.PagedDecoder(path, n_pages=n_pages, max_positions=32, max_seqs=3)
        a, b = d.open(), d.open()
        for t in range(16):
            d.step({a: ids[0][t], b: ids[1][t]})
        return d, a, b

    d, a, b = start(4)
    want = d.step({a: ids[0][16], b: ids[1][16]}), _rows(d, a), _rows(d, b)
    d, a, b = start(4)
    c = d.open()
    d.step({c: 1})
    for status, tokens in ((E.BAD_TOKEN, {a: ids[0][16], b: -1}), (E.OOM, {a: ids[0][16], b: ids[1][16]})):
        for _ in range(3):
            with pytest.raises(E.MCPMError) as e:
                d.step(tokens)
            assert e.value.status == status and len(d.free) == 1 and d.length[a] == d.length[b] == 16
    d.close(c)
    assert d.step({a: ids[0][16], b: ids[1][16]}) == want[0]
    for got, rows in ((_rows(d, a), want[1]), (_rows(d, b), want[2])):
        assert np.array_equal(got[0], rows[0]) and np.array_equal(got[1], rows[1])
    d.close(a), d.close(b)
    assert sorted(d.free) == list(range(4))


@pytest.mark.gpu
def test_a_refused_option_can_be_corrected(cuda, parity):
    """A step whose mask or biases are refused feeds nothing: the corrected one is the undisturbed one."""
    from mcpm import engine as E, paged, synth
    _, _, path = parity
    ids = [int(t) for t in synth.prompt_ids(6, seed=11)]
    options = dict(repetition=1.3, frequency=0.2, presence=0.1, bias={7: 2.0, 130560: 9.0, 2 ** 40: 9.0, -3: 9.0}, allow=np.arange(130560) % 3 > 0)

    def run(disturb):
        d = paged.PagedDecoder(path, n_pages=4, max_positions=32)
        s, out = d.open(), []
        for t in ids:
            if disturb:
                with pytest.raises(ValueError):
                    d.step({s: t}, **{**options, "allow": np.ones(5, bool)})
                with pytest.raises(E.MCPMError):
                    d.step({s: t}, **{**options, "bias": dict.fromkeys(range(5000), 0.0)})
            out.append(d.step({s: t}, **options)[s])
        assert d.history[s] == ids and d.length[s] == d.position[s] == len(ids)
        return out, d.processed[0].cpu().numpy()

    a, b = run(False), run(True)
    assert a[0] == b[0] and np.array_equal(a[1], b[1])


@pytest.mark.gpu
def test_a_conversation_outlives_its_rope_table(cuda, parity):
    """Positions beyond the first table rotate as with one that was long enough."""
    from mcpm import paged, synth
    _, _, path = parity
    ids = [int(t) for t in synth.prompt_ids(60, seed=12)]

    def run(rope_len):
        d = paged.PagedDecoder(path, n_pages=8, max_positions=64, keep=20, slack=16, sink=2, recent=8, rope_len=rope_len)
        s = d.open()
        return [d.step({s: t})[s] for t in ids], d.logits[0].cpu().numpy(), d.k.cpu().numpy()

    a, b = run(4), run(64)
    assert a[0] == b[0] and np.array_equal(a[1], b[1]) and np.array_equal(a[2], b[2])


@pytest.mark.gpu
def test_an_evicting_step_keeps_the_heaviest_of_every_layer(cuda, parity):
    """Masses and rows before a step that evicts name the positions that it keeps: K, V and masses of each layer and KV
    head afterwards, the masses with what the step itself added."""
    from test_gpu_paged import expected_kept
    from mcpm import paged, synth
    _, _, path = parity
    d = paged.PagedDecoder(path, n_pages=8, max_positions=64, keep=30, slack=10, sink=2, recent=8)
    s = d.open()
    evictions = 0
    for t in synth.prompt_ids(75, seed=21):
        n = int(d.length[s])
        if n < 40:
            d.step({s: int(t)})
            continue
        evictions += 1
        page, slot = d.table[s, np.arange(n) // 16].astype(np.int64), np.arange(n) % 16
        k, v, m = (x.cpu().numpy() for x in (d.k, d.v, d.mass))
        d.step({s: int(t)})
        to, at = d.table[s, np.arange(31) // 16].astype(np.int64), np.arange(31) % 16
        k2, v2, m2 = (x.cpu().numpy() for x in (d.k, d.v, d.mass))
        for layer in range(d.n_layer):
            for h in range(2):
                mass = m[layer, page, h, slot]
                kept = expected_kept(mass, np.arange(n), n, 30, 2, 8)
                assert np.array_equal(k2[layer, to[:30], at[:30], h], k[layer, page[kept], slot[kept], h])
                assert np.array_equal(v2[layer, to[:30], at[:30], h], v[layer, page[kept], slot[kept], h])
                now = m2[layer, to, h, at]
                assert np.all(now[:30] >= mass[kept])   # the step adds weights, none below zero
                added = now.astype(np.float64).sum() - mass[kept].astype(np.float64).sum()
                assert abs(added - 8) < 1e-4            # eight heads' weights, over 31 positions, on masses of at most 300
        assert d.length[s] == 31
    assert evictions >= 3
