"""The paged decoder's host side: which steps it refuses, and that a refused step leaves sequences and pages as they
were.  No GPU: every step here is refused before it reaches the device."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")   # mcpm.paged imports it


def decoder(n_pages, max_seqs, lengths, page_size=16, max_positions=64, n_vocab=1000, rope_len=256, **budget):
    """A decoder without weights whose sequences hold the given numbers of positions."""
    from mcpm import paged
    d = paged.PagedDecoder.__new__(paged.PagedDecoder)
    d.page_size, d.max_seqs, d.max_positions, d.n_vocab = page_size, max_seqs, max_positions, n_vocab
    d.keep, d.slack, d.sink, d.recent = (budget.get(k, v) for k, v in dict(keep=0, slack=16, sink=4, recent=16).items())
    d.rope = np.zeros((rope_len, 64, 2), np.float32)
    d.free = list(range(n_pages))[::-1]
    d.table = np.full((max_seqs, max_positions // page_size), -1, np.int32)
    d.length, d.position = np.zeros(max_seqs, np.int32), np.zeros(max_seqs, np.int32)
    d.opened, d.history = [False] * max_seqs, [[] for _ in range(max_seqs)]
    d.evictions = []
    for n in lengths:
        s = d.open()
        for c in range(-(-n // page_size)):
            d.table[s, c] = d._take(1)[0]
        d.length[s] = d.position[s] = n
        d.history[s] = list(range(n))

    def evict(seq):   # what _evict does to the pages
        fresh = np.full(d.table.shape[1], -1, np.int32)
        pages = d._take(-(-d.keep // d.page_size))
        fresh[:len(pages)] = pages
        d._give_back(seq)
        d.table[seq], d.length[seq] = fresh, d.keep
        d.evictions.append(seq)

    d._evict = evict
    return d


def state(d):
    return sorted(d.free), d.table.tolist(), d.length.tolist(), d.position.tolist(), [list(h) for h in d.history], list(d.opened)


def refused(d, status, tokens, **options):
    """status: of an MCPMError, or the exception's type."""
    from mcpm import engine as E
    before = state(d)
    with pytest.raises(status if isinstance(status, type) else E.MCPMError) as e:
        d.step(tokens, **options)
    assert isinstance(status, type) or e.value.status == status
    assert state(d) == before and not d.evictions


def all_pages(d, n_pages):
    for s in range(d.max_seqs):
        d.close(s)
    return sorted(d.free) == list(range(n_pages))


def test_a_refused_step_keeps_no_pages():
    """Two sequences at the end of their pages: whatever stops the second takes no page for the first."""
    from mcpm import engine as E
    d = decoder(5, 2, [16, 32])
    refused(d, E.BAD_TOKEN, {0: 1, 1: 1000})
    refused(d, E.BAD_TOKEN, {0: 1, 1: -1})
    d.opened[1] = False
    refused(d, E.BAD_ARG, {0: 1, 1: 1})
    d.opened[1] = True
    d.length[1] = 64
    refused(d, E.CTX_OVERFLOW, {0: 1, 1: 1})
    d.length[1] = 32
    d.free = d.free[:1]   # one page for two
    refused(d, E.OOM, {0: 1, 1: 1})
    refused(d, E.OOM, {1: 1, 0: 1})
    d.table[1, 2] = d._take(1)[0]   # a page that is there is not taken again
    refused(d, E.OOM, {1: 1, 0: 1})


def test_a_refused_step_evicts_nothing():
    from mcpm import engine as E
    d = decoder(6, 2, [48, 16], keep=32)
    refused(d, E.BAD_TOKEN, {0: 1, 1: 1000})
    d.free = d.free[:1]   # the eviction needs two
    refused(d, E.OOM, {0: 1})
    refused(d, E.OOM, {1: 1, 0: 1})


@pytest.mark.parametrize("order", [(0, 1, 2), (2, 1, 0), (1, 2, 0)])
@pytest.mark.parametrize("free", range(8))
def test_pages_are_counted_in_the_order_of_the_step(order, free):
    """Evictions give pages back that later sequences of the step may take: what _check admits can be carried out, and
    what it refuses cannot."""
    from mcpm import engine as E
    d = decoder(8 + free, 3, [48, 48, 32], keep=32, recent=8)
    other = decoder(8 + free, 3, [48, 48, 32], keep=32, recent=8)

    try:
        evicted = d._check({s: 1 for s in order})
    except E.MCPMError as e:
        assert e.status == E.OOM
        with pytest.raises(E.MCPMError):
            other._admit(order, [0, 1])
        return
    assert evicted == [s for s in order if s < 2]
    d._admit(order, evicted)
    assert d.evictions == evicted and all_pages(d, 8 + free)


def test_a_refused_option_feeds_no_token():
    """Masks of the wrong shape, too many biases and penalties that mean nothing are found before the step begins."""
    from mcpm import engine as E
    d = decoder(6, 2, [48, 16], keep=32)
    t = {0: 1, 1: 2}
    refused(d, ValueError, t, allow=np.ones(999, bool))
    refused(d, ValueError, t, allow=np.ones((3, 1000), bool))
    refused(d, E.BAD_ARG, t, bias={i: 1.0 for i in range(E.MAX_BIAS + 1)})
    for r in (0.0, -1.0, float("nan")):
        refused(d, E.BAD_ARG, t, repetition=r)
    refused(d, TypeError, {0: 1, 1: 2.5})


def test_limits_are_the_operators_own():
    from mcpm import engine as E
    lib = E.load_library()
    for more in (dict(hist=256, penalties=256, hist_max=E.MAX_HIST + 1), dict(bias_token=256, bias=256, bias_max=E.MAX_BIAS + 1)):
        p = E.mcpm_logits_params(n_seq=1, n_vocab=100, logits=256, out=512, **more)
        assert lib.mcpm_logits_process(p, None) == E.BAD_ARG


def test_sequence_numbers_are_not_indexes_from_the_end():
    """-1 names no sequence: with 1 it would feed two tokens to one slot of the last."""
    from mcpm import engine as E
    d = decoder(6, 2, [3, 5])
    for tokens in ({-1: 1}, {1: 1, -1: 2}, {0: 1, 2: 1}):
        refused(d, E.BAD_ARG, tokens)
    refused(d, TypeError, {0.5: 1})
    before = state(d)
    for s in (-1, 2):
        with pytest.raises(E.MCPMError) as e:
            d.close(s)
        assert e.value.status == E.BAD_ARG and state(d) == before
    d.close(1)
    d.close(1)   # an unused one: nothing to do
    assert len(d.free) == 5


@pytest.mark.parametrize("budget", [dict(slack=-1), dict(slack=-32), dict(sink=-1), dict(recent=-1, sink=20), dict(keep=-1), dict(keep=64, slack=0),
                                    dict(slack=33), dict(sink=30, recent=3)])
def test_budgets_that_cannot_be_kept(budget):
    """With a negative slack a sequence was cut to `keep` positions while it still had fewer, and attended to slots that
    nothing had been written to.  Refused before the file is opened."""
    from mcpm import paged
    with pytest.raises(ValueError) as e:
        paged.PagedDecoder("no such file", n_pages=8, max_positions=64, **{**dict(keep=32, sink=2, recent=8), **budget})
    assert "keep" in str(e.value)


def write_header(path, change=lambda t: t, short=0):
    """A model file without weights: the header, and a hole of the data section's size less `short` bytes."""
    from mcpm import spec, synth
    tensors = [t for t in map(change, spec.tensor_list("q4_k_m")) if t is not None and (not t.name.startswith("blk.") or t.name.startswith("blk.0."))]
    tensors = spec.layout(tensors, spec.Q4KM_DATA_START)
    with open(path, "wb") as f:
        f.write(synth._header(tensors, spec.Q4KM_DATA_START, "q4_k_m"))
        f.truncate(tensors[-1].offset + tensors[-1].nbytes - short)
    return str(path)


def test_model_file(tmp_path):
    from mcpm import paged, spec
    tensors, n_layer = paged.model_tensors(write_header(tmp_path / "m.gguf"))
    assert n_layer == 1 and len(tensors) == 3 + len(spec.LAYER_TENSORS)
    assert tensors["blk.0.ffn_down.weight"].dims == (spec.N_FF, spec.N_EMBD)


@pytest.mark.parametrize("name,dims,kind,status", [
    ("blk.0.ffn_gate.weight", (2048, 8192), 12, "BAD_FILE"), ("blk.0.ffn_down.weight", (8192, 2048), 14, "BAD_FILE"),
    ("blk.0.attn_k.weight", (2048, 2048), 12, "BAD_FILE"), ("output.weight", (2048, 131072), 14, "BAD_FILE"),
    ("blk.0.attn_norm.weight", (1024,), 0, "BAD_FILE"), ("token_embd.weight", (4096, 130560), 12, "BAD_FILE"),
    ("blk.0.attn_v.weight", None, 12, "BAD_FILE"), ("blk.0.attn_q.weight", None, 12, "BAD_FILE"), ("output_norm.weight", None, 0, "BAD_FILE"),
    ("token_embd.weight", (2048, 130560), 14, "UNSUPPORTED_TYPE"), ("blk.0.attn_q.weight", (2048, 2048), 8, "UNSUPPORTED_TYPE"),
    ("blk.0.ffn_norm.weight", (2048,), 1, "UNSUPPORTED_TYPE")])
def test_models_of_another_shape_are_refused(tmp_path, name, dims, kind, status):
    """Wider layers would have written beyond the decoder's buffers.  Refused before anything is uploaded."""
    from mcpm import engine as E, paged, spec
    path = write_header(tmp_path / "m.gguf", lambda t: t if t.name != name else dims and spec.TensorInfo(name, kind, dims))
    with pytest.raises(E.MCPMError) as e:
        paged.PagedDecoder(path, n_pages=4)
    assert e.value.status == getattr(E, status)


def test_a_truncated_model_is_refused(tmp_path):
    """The last tensor's missing bytes would have been read beyond its copy on the device."""
    from mcpm import engine as E, paged
    with pytest.raises(E.MCPMError) as e:
        paged.PagedDecoder(write_header(tmp_path / "m.gguf", short=1), n_pages=4)
    assert e.value.status == E.BAD_FILE


def test_positions_count_beyond_the_first_rope_table():
    """A sequence whose cache is bounded does not end where the table of rotations did."""
    d = decoder(6, 2, [10, 20], keep=32, rope_len=30)
    d.position[:] = [10, 30]
    assert d._check({0: 1, 1: 1}) == []
    made = []
    d._rope_table = lambda n: made.append(n) or np.zeros((n, 64, 2), np.float32)
    for p in (10, 29, 30, 59, 60, 500):
        d._reach(p)
        assert d.rope.shape[0] > p
    assert made == [60, 120, 501]


def test_histories_beyond_the_operators_limit():
    """Penalties count the last tokens that the operator takes; a long conversation is not refused."""
    from mcpm import engine as E
    d = decoder(6, 2, [16, 16])
    d._dev = lambda a, dtype=np.int32: torch.from_numpy(np.ascontiguousarray(a, dtype=dtype))
    d.history = [[3] * 5 + [4] * (E.MAX_HIST - 1), [5, 6]]
    held, more = d._options({0: 9, 1: 8}, 1.1, 0.0, 0.0, None, None)
    hist = held[0].numpy()
    assert hist.shape == (2, E.MAX_HIST) and more["hist_stride"] == E.MAX_HIST
    assert (hist[0, :-1] == 4).all() and hist[0, -1] == 9
    assert hist[1, :3].tolist() == [5, 6, 8] and (hist[1, 3:] == -1).all()


@pytest.mark.parametrize("page_size,keep,slack", [(16, 32, 16), (16, 20, 0), (16, 33, 5), (7, 40, 3), (1, 20, 7)])
def test_the_stated_pages_are_enough(page_size, keep, slack):
    """Sequences at their budgets in one pool, stepped together in any order, never run out of pages."""
    n = 3 * -(-(keep + max(slack, 1)) // page_size) + -(-keep // page_size)
    d = decoder(n, 3, [0, 0, 0], page_size=page_size, max_positions=-(-(keep + slack + 1) // page_size) * page_size, keep=keep, slack=slack,
                sink=2, recent=8)
    rng = np.random.default_rng(page_size)
    for _ in range(400):
        seqs = [int(s) for s in rng.permutation(3)[:rng.integers(1, 4)]]
        d._admit(seqs, d._check({s: 1 for s in seqs}))
        d.length[seqs] += 1
        assert len(d.free) + int((d.table >= 0).sum()) == n
    assert d.evictions and all_pages(d, n)
