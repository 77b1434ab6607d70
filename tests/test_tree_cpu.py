"""CPU: host logic and refusals of the tree-verification operators."""
import ctypes
import math

import numpy as np
import pytest
import torch


def _up(parents, i):
    seen = [i]
    while parents[seen[-1]] >= 0:
        seen.append(parents[seen[-1]])
    return seen


@pytest.mark.parametrize("T", [1, 2, 7, 31, 64])
def test_draft_tree_masks_follow_the_parents(dsa, T):
    rng = np.random.default_rng(T)
    parents = np.stack([np.array([rng.integers(-1, i) if i else -1 for i in range(T)]),
                        np.arange(T) - 1,            # a line: depth grows by one, log2 T doublings are needed
                        np.full(T, -1)])             # all roots
    mask, depth = dsa.mla_sparse.draft_tree_masks(torch.tensor(parents, dtype=torch.int32))
    for b in range(3):
        for i in range(T):
            path = _up(parents[b], i)
            want = sum(1 << int(j) for j in path)
            assert int(mask[b, i]) & (2 ** 64 - 1) == want, (b, i)
            assert int(depth[b, i]) == len(path) - 1


def test_draft_tree_masks_take_bad_parents_as_roots(dsa):
    mask, depth = dsa.mla_sparse.draft_tree_masks(torch.tensor([[3, 5, 2, -9]]))
    assert mask.tolist() == [[1, 2, 4, 8]] and depth.tolist() == [[0, 0, 0, 0]]
    mask, depth = dsa.mla_sparse.draft_tree_masks(torch.empty(2, 0, dtype=torch.int32))
    assert mask.shape == (2, 0) and depth.shape == (2, 0)
    with pytest.raises(RuntimeError, match="64 drafts"):
        dsa.mla_sparse.draft_tree_masks(torch.zeros(1, 65, dtype=torch.int32))


def test_rope_table_without_scaling_and_far_positions(dsa):
    t = dsa.rope.rope_cos_sin_cache(64, 180_001, base=1e6)
    p, i = 180_000, np.arange(32)
    a = np.float64(p) * 1e6 ** (-2.0 * i / 64)
    # one rounding to f32 of a value of at most 1, and f64's error of an angle below 2e5 (2^-53 * 2e5)
    assert np.abs(t[p, :32].double().numpy() - np.cos(a)).max() <= 2.0 ** -24 + 1e-10
    assert np.abs(t[p, 32:].double().numpy() - np.sin(a)).max() <= 2.0 ** -24 + 1e-10


def test_rope_table_scalings(dsa):
    r = dsa.rope
    plain, g = r.rope_inv_freq(64)
    assert g == 1.0
    lin, _ = r.rope_inv_freq(64, scaling={"type": "linear", "factor": 4.0})
    assert torch.equal(lin, plain / 4.0)
    ntk, _ = r.rope_inv_freq(64, scaling={"type": "ntk", "factor": 8.0})
    assert ntk[0] == 1.0 and abs(float(ntk[31] / plain[31]) - 1 / 8.0) < 1e-12  # last pair: wavelength times the factor
    y, g = r.rope_inv_freq(64, scaling={"type": "yarn", "factor": 40.0, "original_max_position": 4096})
    assert abs(g - (0.1 * math.log(40.0) + 1.0)) < 1e-12
    turns = 4096 * plain / (2 * math.pi)
    # floor / ceil widen the ramp to whole pairs: one pair past the thresholds all is kept / divided
    assert torch.equal(y[turns > 32 * 10000 ** (2 / 64)], plain[turns > 32 * 10000 ** (2 / 64)])
    assert torch.allclose(y[turns < 1], plain[turns < 1] / 40.0, rtol=1e-14, atol=0)
    mid = (y < plain) & (y > plain / 40.0)
    assert 5 < int(mid.sum()) < 20 and bool((y[1:] < y[:-1]).all())
    same, g = r.rope_inv_freq(64, scaling={"type": "yarn", "factor": 40.0, "original_max_position": 4096,
                                           "mscale": 1.0, "mscale_all_dim": 1.0})
    assert g == 1.0 and torch.equal(same, y)
    for bad in ({"type": "no"}, {"type": "linear", "factor": 0.0}):
        with pytest.raises(RuntimeError):
            r.rope_inv_freq(64, scaling=bad)
    with pytest.raises(RuntimeError):
        r.rope_inv_freq(63)
    with pytest.raises(RuntimeError):
        r.rope_cos_sin_cache(64, 0)


def _ops(dsa):
    return dsa.ops


def test_wrappers_refuse_cpu_tensors(dsa):
    ops = _ops(dsa)
    i32 = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops._tree_mla_decode_impl(torch.empty(1, 1, 1, 512), torch.empty(1, 1, 1), torch.empty(1, 1, 1, 576),
                                  torch.empty(1, 64, 576), i32[None], i32, torch.zeros(1, 1, dtype=torch.int64), None, 1.0)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops._commit_draft_rows_impl([torch.empty(1, 64, 576)], i32[None], i32, i32[None], i32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops._gather_cache_impl(torch.empty(1, 576), torch.empty(1, 64, 576), i32[None], i32, None)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops._rotary_embedding_impl(torch.empty(1, 1, 64), torch.empty(1, 1, 64), torch.zeros(1, dtype=torch.int64),
                                   torch.empty(1, 64), False, 0)
    ops._commit_draft_rows_impl([], i32[None], i32, i32[None], i32)  # nothing to do


def _tree(lib, **k):
    P = ctypes.c_void_p
    a = dict(o=P(1024), o_dtype=1, lse=P(1024), q=P(1024), q_dtype=1, kv=P(1024), fmt=3, n_rows=640, page=64, bt=P(1024),
             bts=4, mb=4, seq=P(1024), dl=None, mask=P(1024), ms=8, B=1, T=8, H=8, scale=1.0, ws=None, wsb=0, stream=None)
    a.update(k)
    return lib.dsa_tree_mla_decode(*a.values())


def test_tree_entry_refuses_bad_arguments(dsa):
    L, lib = dsa._lib, dsa._lib.lib()
    P = ctypes.c_void_p
    for bad, code in [(dict(B=-1), L.DSA_ERR_INVALID), (dict(T=65, ms=65), L.DSA_ERR_UNSUPPORTED),
                      (dict(q_dtype=2), L.DSA_ERR_INVALID), (dict(o_dtype=2), L.DSA_ERR_INVALID),
                      (dict(fmt=4), L.DSA_ERR_INVALID), (dict(fmt=1, q_dtype=0), L.DSA_ERR_UNSUPPORTED),
                      (dict(page=0), L.DSA_ERR_INVALID), (dict(n_rows=2 ** 31), L.DSA_ERR_INVALID),
                      (dict(bts=3), L.DSA_ERR_INVALID), (dict(ms=7), L.DSA_ERR_INVALID), (dict(q=None), L.DSA_ERR_INVALID),
                      (dict(mask=None), L.DSA_ERR_INVALID), (dict(bt=None), L.DSA_ERR_INVALID),
                      (dict(kv=P(1032)), L.DSA_ERR_INVALID), (dict(o=P(1032)), L.DSA_ERR_INVALID),
                      (dict(H=2000), L.DSA_ERR_UNSUPPORTED)]:
        assert _tree(lib, **bad) == code, bad
    assert _tree(lib, B=0) == L.DSA_OK and _tree(lib, T=0) == L.DSA_OK and _tree(lib, H=0) == L.DSA_OK


def test_rotary_entry_refuses_bad_arguments(dsa):
    L, lib = dsa._lib, dsa._lib.lib()
    P = ctypes.c_void_p

    def call(**k):
        a = dict(out=P(1024), ot=64, oh=64, x=P(1024), xt=64, xh=64, dt=1, pos=P(1024), cs=P(1024), mp=10, r=64, off=0,
                 neox=0, n=4, h=1, w=64, s=None)
        a.update(k)
        return lib.dsa_rotary_embedding(*a.values())

    for bad, code in [(dict(dt=3), L.DSA_ERR_INVALID), (dict(r=63), L.DSA_ERR_INVALID), (dict(r=0), L.DSA_ERR_INVALID),
                      (dict(off=1), L.DSA_ERR_INVALID), (dict(off=-2), L.DSA_ERR_INVALID), (dict(n=-1), L.DSA_ERR_INVALID),
                      (dict(mp=0), L.DSA_ERR_INVALID), (dict(x=None), L.DSA_ERR_INVALID), (dict(w=0), L.DSA_ERR_INVALID),
                      (dict(w=4096), L.DSA_ERR_UNSUPPORTED), (dict(h=70000), L.DSA_ERR_UNSUPPORTED)]:
        assert call(**bad) == code, bad
    assert call(n=0) == L.DSA_OK and call(h=0) == L.DSA_OK


def test_rotary_entry_refuses_heads_that_overlap(dsa):
    """Strides of out that give two heads the same element; x may repeat its heads."""
    L, lib = dsa._lib, dsa._lib.lib()
    P = ctypes.c_void_p

    def call(n, h, ot, oh):
        return lib.dsa_rotary_embedding(P(1024), ot, oh, P(1024), 0, 0, 1, P(1024), P(1024), 10, 64, 0, 0, n, h, 64, None)

    for n, h, ot, oh in [(4, 1, 0, 64), (4, 1, 63, 0), (1, 3, 0, 0), (1, 3, 999, 56), (4, 3, 64, 64), (4, 3, 128, 64),
                         (4, 3, 64, 192), (4, 3, 191, 64), (4, 3, -192, 64), (2, 2, 1 << 62, 1 << 62)]:
        assert call(n, h, ot, oh) == L.DSA_ERR_INVALID, (n, h, ot, oh)


def test_sizes_beyond_32_bits_are_refused(dsa):
    dsa.ops._fits(1, (1 << 31) - 1)
    with pytest.raises(RuntimeError, match="2.31"):
        dsa.ops._fits(3, 1 << 31)


def test_gather_and_commit_entries_refuse_bad_arguments(dsa):
    L, lib = dsa._lib, dsa._lib.lib()
    P = ctypes.c_void_p

    def gather(**k):
        a = dict(out=P(1024), od=1, os=576, n=4, c=P(1024), fmt=3, rows=640, page=64, w=576, bt=P(1024), bts=4, mb=4,
                 cu=P(1024), st=None, B=1, s=None)
        a.update(k)
        return lib.dsa_gather_cache(*a.values())

    for bad in [dict(od=2), dict(fmt=2), dict(w=128), dict(fmt=4), dict(fmt=0, w=20, os=24), dict(n=-1), dict(page=0),
                dict(bts=3), dict(os=512), dict(os=580), dict(out=P(1028)), dict(c=P(1028)), dict(cu=None),
                dict(bt=None), dict(c=None)]:
        assert gather(**bad) == L.DSA_ERR_INVALID, bad
    assert gather(n=0) == L.DSA_OK and gather(B=0) == L.DSA_OK

    def commit(ptrs=(1024,), **k):
        arr = (ctypes.c_void_p * max(1, len(ptrs)))(*ptrs)
        a = dict(c=arr, nc=len(ptrs), rows=640, page=64, rb=656, bt=P(1024), bts=4, mb=4, seq=P(1024), dl=P(1024), nd=64,
                 acc=P(1024), acs=8, na=8, B=1, s=None)
        a.update(k)
        return lib.dsa_commit_draft_rows(*a.values())

    for bad, code in [(dict(nd=65), L.DSA_ERR_UNSUPPORTED), (dict(na=65, acs=65), L.DSA_ERR_UNSUPPORTED),
                      (dict(rb=654), L.DSA_ERR_UNSUPPORTED), (dict(rb=1168), L.DSA_ERR_UNSUPPORTED),
                      (dict(rb=260), L.DSA_ERR_UNSUPPORTED), (dict(acs=7), L.DSA_ERR_INVALID), (dict(B=-1), L.DSA_ERR_INVALID),
                      (dict(acc=None), L.DSA_ERR_INVALID), (dict(ptrs=(1028,)), L.DSA_ERR_INVALID),
                      (dict(ptrs=(1024, 0)), L.DSA_ERR_INVALID)]:
        assert commit(**bad) == code, bad
    assert commit(ptrs=()) == L.DSA_OK and commit(B=0) == L.DSA_OK and commit(na=0) == L.DSA_OK


def test_new_ops_registered(dsa):
    ns = torch.ops.dsa_b200
    assert [a.name for a in ns.tree_mla_decode.default._schema.arguments] == [
        "o", "lse", "q", "kv_cache", "block_table", "seq_lens", "tree_mask", "draft_lens", "scale"]
    for name in ("tree_mla_decode", "commit_draft_rows", "gather_cache", "rotary_embedding"):
        assert hasattr(ns, name) and callable(getattr(dsa, name))


def test_expanded_rows_keep_their_stride(dsa):
    """One tree, path or table row shared by a batch (expand) has a row stride of 0:
    the entry points get that, not the width, which would take them past its storage."""
    ops, L, lib = _ops(dsa), dsa._lib, dsa._lib.lib()
    one = torch.arange(3, dtype=torch.int32)[None]
    assert ops._pages(one.expand(4, 3), 4)[1:] == (0, 3)
    assert ops._pages(one, 1)[1:] == (3, 3)
    assert ops._pages(torch.as_strided(one, (1, 3), (1, 1)), 1)[1:] == (3, 3)  # one row: any stride
    assert ops._pages(torch.zeros(4, 9, dtype=torch.int32)[:, 2:5], 4)[1:] == (9, 3)
    assert ops._pages(torch.as_strided(torch.zeros(9, dtype=torch.int32), (4, 3), (2, 1)), 4)[1:] == (2, 3)
    # the entries take 0 and what rows that do not overlap have, nothing between
    P = ctypes.c_void_p
    for stride, code in [(0, L.DSA_OK), (4, L.DSA_OK), (9, L.DSA_OK), (1, L.DSA_ERR_INVALID), (3, L.DSA_ERR_INVALID),
                         (-4, L.DSA_ERR_INVALID)]:
        assert _tree(lib, B=0, bts=stride) == code, stride
        assert _tree(lib, B=0, T=4, ms=stride) == code, stride
        assert lib.dsa_gather_cache(P(1024), 1, 576, 4, P(1024), 3, 640, 64, 576, P(1024), stride, 4, P(1024), None, 0,
                                    None) == code, stride
        caches = (ctypes.c_void_p * 1)(1024)
        assert lib.dsa_commit_draft_rows(caches, 1, 640, 64, 656, P(1024), 4, 4, P(1024), P(1024), 64, P(1024), stride, 4, 0,
                                         None) == code, stride


def test_commit_entry_refuses_one_table_row_for_several_requests(dsa):
    L, lib = dsa._lib, dsa._lib.lib()
    P = ctypes.c_void_p

    def call(B, bts, rows=0):
        return lib.dsa_commit_draft_rows((ctypes.c_void_p * 1)(1024), 1, rows, 64, 656, P(1024), bts, 4, P(1024), P(1024),
                                         64, P(1024), 8, 8, B, None)

    assert call(2, 0, rows=640) == L.DSA_ERR_INVALID
    assert call(1, 0) == L.DSA_OK and call(2, 4) == L.DSA_OK  # (a cache without rows: nothing to move)


def test_tree_wrapper_rounds_queries_to_the_cache_type(dsa, monkeypatch):
    """What forward_mqa_tree hands to the operator, for each type of q and cache."""
    seen = {}
    monkeypatch.setattr(dsa.ops, "tree_mla_decode", lambda o, lse, q, kv, bt, ln, mask, scale, dl: seen.update(
        o=o.dtype, q=q.dtype, bt=bt.dtype, ln=ln.dtype, dl=None if dl is None else dl.dtype))
    bf, hf, f32, i32, i64 = torch.bfloat16, torch.float16, torch.float32, torch.int32, torch.int64
    for q, kv, want in [(f32, bf, bf), (f32, hf, hf), (f32, torch.uint8, hf), (torch.float64, bf, bf), (bf, hf, bf),
                        (hf, torch.uint8, hf), (bf, torch.uint8, bf)]:
        for lens in (None, torch.ones(1, dtype=i64), torch.ones(1, dtype=i32)):
            o, lse = dsa.mla_sparse.forward_mqa_tree(torch.zeros(1, 2, 3, 576, dtype=q), torch.zeros(1, 64, 576).to(kv),
                                                     torch.zeros(1, 1, dtype=i64), torch.ones(1, dtype=i64),
                                                     torch.ones(1, 2, dtype=i64), 1.0, draft_lens=lens)
            assert seen == dict(o=want, q=want, bt=i32, ln=i32, dl=None if lens is None else i32)
            assert o.dtype == want and o.shape == (1, 2, 3, 512) and lse.shape == (1, 2, 3)


def test_tree_entry_refuses_scales_that_f32_cannot_hold(dsa):
    """A finite double beyond f32 would make every score infinite or NaN."""
    L, lib = dsa._lib, dsa._lib.lib()
    for scale in (1e39, -1e300, 3e38, math.inf, -math.inf, math.nan):  # 3e38 log2(e) is past f32's 3.4e38
        assert _tree(lib, B=0, scale=scale) == L.DSA_ERR_INVALID, scale
    for scale in (0.0, -1.0, 1e-320, 1e30):
        assert _tree(lib, B=0, scale=scale) == L.DSA_OK, scale


def test_rotary_entry_refuses_an_out_that_overlaps_x(dsa):
    """Every shift of x against out, with strides in both orders, against sets of
    elements. Calls that are to be served have no table, which is refused later on."""
    L, lib = dsa._lib, dsa._lib.lib()
    P = ctypes.c_void_p

    def refused(n, h, st, sh, w, shift):
        lib.dsa_rotary_embedding(P(1 << 20), st, sh, P((1 << 20) - 2 * shift), st, sh, 1, P(1024), P(1024), 0, 4, 0, 0, n, h, w,
                                 None)
        return b"overlaps x" in lib.dsa_last_error()

    for n, h, st, sh, w in [(3, 4, 40, 9, 8), (3, 4, 9, 30, 8), (1, 3, 5, 16, 4), (4, 1, 6, 77, 6), (1, 1, 0, 0, 8), (2, 2, 64, 32, 8)]:
        heads = {t * (st if n > 1 else 0) + k * (sh if h > 1 else 0) + e for t in range(n) for k in range(h) for e in range(w)}
        for shift in range(-170, 171):
            meet = shift != 0 and any(p - shift in heads for p in heads)
            assert refused(n, h, st, sh, w, shift) == meet, (n, h, st, sh, w, shift)
