"""Refusals of the paged KV-cache calls (no GPU: every call is refused before it reaches the device) and the
RoPE table, which is computed on the host."""
import numpy as np
import pytest

A = 256   # an aligned address that is never dereferenced


def config(E, **change):
    c = E.paged_config(E.KV_F16, 16, 2, 128, 16, 100, 8, 32)
    for k, v in change.items():
        setattr(c, k, v)
    return c


BAD_CONFIGS = [dict(n_head=0), dict(n_head_kv=0), dict(n_head=15), dict(n_head=34), dict(n_head=-16), dict(head_dim=96),
               dict(head_dim=0), dict(page_size=0), dict(page_size=-1), dict(n_pages=0), dict(max_seqs=0), dict(max_seqs=65536),
               dict(max_pages=0), dict(n_pages=1 << 28), dict(max_pages=1 << 27), dict(page_stride=4096), dict(page_stride=4096, row_stride=4, head_stride=128),
               dict(page_stride=-4096, row_stride=256, head_stride=128)]


@pytest.mark.parametrize("change", BAD_CONFIGS)
def test_bad_configurations(change):
    from mcpm import engine as E
    lib = E.load_library()
    c, pool, tok = config(E, **change), E.paged_pool(A, A, A), E.mcpm_paged_tokens(n_tok=1, tok_slot=A, k=A, v=A)
    assert lib.mcpm_paged_workspace_bytes(c) == 0
    with pytest.raises(E.MCPMError):
        E.paged_workspace_bytes(c)
    assert lib.mcpm_paged_append(c, pool, A, 1, tok, None) == E.BAD_ARG
    assert lib.mcpm_paged_attention(c, pool, A, A, 1, A, 0, A, 0.0, A, 1 << 40, None) == E.BAD_ARG
    assert lib.mcpm_paged_evict(c, pool, A, A, 2 * A, A, A, 1, 4, 0, 0, A, 1 << 40, None) == E.BAD_ARG


def test_unsupported_type():
    from mcpm import engine as E
    lib = E.load_library()
    c = config(E, kv_type=3)
    assert lib.mcpm_paged_workspace_bytes(c) == 0
    assert lib.mcpm_paged_attention(c, E.paged_pool(A, A), A, A, 1, A, 0, A, 0.0, A, 1 << 40, None) == E.UNSUPPORTED_TYPE


@pytest.mark.parametrize("pool", [(0, A), (A, 0), (A + 8, A), (A, A + 2)])
def test_bad_pools(pool):
    from mcpm import engine as E
    lib = E.load_library()
    c, p = config(E), E.mcpm_paged_pool(pool[0] or None, pool[1] or None, A)
    assert lib.mcpm_paged_append(c, p, A, 1, E.mcpm_paged_tokens(n_tok=1, tok_slot=A, k=A, v=A), None) == E.BAD_ARG
    assert lib.mcpm_paged_attention(c, p, A, A, 1, A, 0, A, 0.0, A, 1 << 40, None) == E.BAD_ARG
    assert lib.mcpm_paged_evict(c, p, A, A, 2 * A, A, A, 1, 4, 0, 0, A, 1 << 40, None) == E.BAD_ARG


@pytest.mark.parametrize("change", [
    dict(n_tok=-1), dict(tok_slot=None), dict(k=None), dict(v=None), dict(k=A + 4), dict(v=A + 8), dict(kv_stride=128), dict(kv_stride=258),
    dict(q=A), dict(q=A + 4, q_out=A), dict(q=A, q_out=A + 4), dict(q=A, q_out=2 * A, q_stride=1024), dict(q=A, q_out=2 * A, q_stride=2050),
    dict(q=A, q_out=A, q_stride=2560), dict(rope=A), dict(rope=A, rope_len=-1), dict(rope=A + 8, rope_len=4)])
def test_append_refusals(change):
    from mcpm import engine as E
    lib = E.load_library()
    t = E.mcpm_paged_tokens(n_tok=1, tok_slot=A, k=A, v=A)
    for k, v in change.items():
        setattr(t, k, v)
    assert lib.mcpm_paged_append(config(E), E.paged_pool(A, A), A, 1, t, None) == E.BAD_ARG
    assert lib.mcpm_paged_append(config(E), E.paged_pool(A, A), A, 9, E.mcpm_paged_tokens(n_tok=1, tok_slot=A, k=A, v=A), None) == E.BAD_ARG
    assert lib.mcpm_paged_append(config(E), E.paged_pool(A, A), None, 1, E.mcpm_paged_tokens(n_tok=1, tok_slot=A, k=A, v=A), None) == E.BAD_ARG
    assert lib.mcpm_paged_append(config(E), E.paged_pool(A, A), A, 1, None, None) == E.BAD_ARG
    assert lib.mcpm_paged_append(None, E.paged_pool(A, A), A, 1, E.mcpm_paged_tokens(n_tok=1, tok_slot=A, k=A, v=A), None) == E.BAD_ARG


GOOD = dict(table=A, len=A, n=1, q=A, q_stride=0, out=A, scale=0.0, ws=A, bytes=1 << 40)


@pytest.mark.parametrize("change", [
    dict(table=None), dict(len=None), dict(n=0), dict(n=9), dict(q=None), dict(q=A + 4), dict(q_stride=2047), dict(q_stride=2050), dict(out=None),
    dict(out=A + 8), dict(scale=-1.0), dict(scale=float("nan")), dict(ws=None), dict(ws=A + 8), dict(bytes=0)])
def test_attention_refusals(change):
    from mcpm import engine as E
    a = {**GOOD, **change}
    st = E.load_library().mcpm_paged_attention(config(E), E.paged_pool(A, A), a["table"], a["len"], a["n"], a["q"], a["q_stride"], a["out"],
                                               a["scale"], a["ws"], a["bytes"], None)
    assert st == E.BAD_ARG


@pytest.mark.parametrize("change", [
    dict(mass=0), dict(table=None), dict(len=None), dict(dst=None), dict(dst=A), dict(new_len=None), dict(kept=None), dict(n=0), dict(n=9), dict(keep=0),
    dict(keep=513), dict(sink=-1), dict(recent=-1), dict(sink=5), dict(sink=2, recent=3), dict(recent=2 ** 31 - 1, sink=2), dict(ws=None), dict(bytes=8)])
def test_evict_refusals(change):
    from mcpm import engine as E
    a = {**dict(mass=A, table=A, len=A, dst=2 * A, new_len=A, kept=A, n=1, keep=4, sink=0, recent=0, ws=A, bytes=1 << 40), **change}
    st = E.load_library().mcpm_paged_evict(config(E), E.paged_pool(A, A, a["mass"]), a["table"], a["len"], a["dst"], a["new_len"], a["kept"], a["n"],
                                           a["keep"], a["sink"], a["recent"], a["ws"], a["bytes"], None)
    assert st == E.BAD_ARG


def test_rope_table():
    from mcpm import engine as E
    t = E.rope_table(50, 128, 10000.0)
    angle = np.arange(50)[:, None] * 10000.0 ** (-np.arange(0, 128, 2) / 128)
    # fp32 theta and angle: relative errors of a few 2^-24, the angle at most 49
    assert np.allclose(t[..., 0], np.cos(angle), atol=49 * 2.0 ** -21) and np.allclose(t[..., 1], np.sin(angle), atol=49 * 2.0 ** -21)
    lib = E.load_library()
    assert lib.mcpm_rope_table(None, 4, 128, 1e4) == E.BAD_ARG
    buf = np.zeros(8, np.float32)
    for n, d, base in ((0, 2, 1e4), (4, 3, 1e4), (4, 0, 1e4), (4, 2, 0.0), (4, 2, float("nan"))):
        assert lib.mcpm_rope_table(E._fptr(buf), n, d, base) == E.BAD_ARG


def test_cluster_width_rules(tmp_path):
    """Clusters of 16 CTAs where the device can run one, of the portable 8 elsewhere, and no question asked up to 8."""
    import os
    import subprocess
    from conftest import PKG, REPO
    exe = str(tmp_path / "cluster_width")
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(PKG, "csrc"), os.path.join(REPO, "tests", "cpp", "cluster_width.cpp"), "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, check=True).stdout
    assert [int(x) for x in out.split()] == [16, 8, 8, 8, 1, 3, 130, 116, 7]
