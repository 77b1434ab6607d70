"""GPU: the tree-verification operators against plain 64-bit implementations."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
SCALE = 192 ** -0.5
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def make_cache(fmt, pages, page, seed, oracle):
    """Cache tensor of N(0, 1) rows."""
    x = torch.randn(pages * page, 576, generator=gen(seed), device=DEV)
    if fmt == "fp8":
        raw = torch.empty(pages * page, 656, dtype=torch.uint8, device=DEV)
        s = x[:, :512].view(-1, 4, 128).abs().amax(2) / 448.0
        raw[:, :512] = (x[:, :512].view(-1, 4, 128) / s[..., None]).to(torch.float8_e4m3fn).view(torch.uint8).view(-1, 512)
        raw[:, 512:528] = s.contiguous().view(torch.uint8).view(-1, 16)
        raw[:, 528:] = x[:, 512:].half().contiguous().view(torch.uint8).view(-1, 128)
        return raw.view(pages, page, 656)
    return x.to(HF if fmt == "f16" else BF).view(pages, page, 576)


def values64(cache):
    rows = cache.reshape(-1, cache.shape[-1])
    if cache.dtype != torch.uint8:
        return rows.double()
    code = rows[:, :512].contiguous().view(torch.float8_e4m3fn).double().view(-1, 4, 128)
    scale = rows[:, 512:528].contiguous().view(F32).double()
    return torch.cat([(code * scale[..., None]).view(-1, 512), rows[:, 528:].contiguous().view(HF).double()], 1)


def tree64(q, cache, table, lens, mask, drafts, scale):
    """o, lse, and per row the largest sum_d |q_d k_d| * scale over the seen
    positions and sum_p p |v|, which the error bounds are made of."""
    B, T, H, _ = q.shape
    kv_all, page = values64(cache), cache.shape[-2]
    o = torch.zeros(B, T, H, 512, dtype=torch.float64, device=DEV)
    mag = torch.zeros_like(o)
    lse = torch.full((B, T, H), -np.inf, dtype=torch.float64, device=DEV)
    zmag = torch.zeros(B, T, H, dtype=torch.float64, device=DEV)
    for b in range(B):
        n = T if drafts is None else min(max(int(drafts[b]), 0), T)
        s = int(lens[b])
        for i in range(n):
            bits = int(mask[b, i])
            pos = [p for p in range(max(s - n, 0))] + [s - n + j for j in range(n) if bits >> j & 1 and s - n + j >= 0]
            if not pos:
                continue
            pos = torch.tensor(pos, device=DEV)
            blk = pos // page
            ok = blk < table.shape[1]
            row = table[b].long()[blk.clamp(max=table.shape[1] - 1)] * page + pos % page
            ok &= (row >= 0) & (row < kv_all.shape[0])
            kv = torch.where(ok[:, None], kv_all[row.clamp(0, kv_all.shape[0] - 1)], 0.0)
            x = q[b, i].double()
            z = x @ kv.t() * scale
            lse[b, i] = torch.logsumexp(z, 1)
            p = torch.exp(z - lse[b, i][:, None])
            o[b, i], mag[b, i] = p @ kv[:, :512], p @ kv[:, :512].abs()
            zmag[b, i] = (x.abs() @ kv.abs().t()).amax(1) * abs(scale)
    return o, lse, zmag, mag


def check_tree(got_o, got_lse, ref, fmt):
    """Elementwise: a score is off by at most zmag times half an fp16 step of
    the key (2^-11, fp8 caches only: 16-bit rows and q enter the product
    exactly) and 2^-24 per term of an f32 sum of 576; the probabilities and the
    dequantised values are rounded once (2^-11; bf16 caches: probabilities to
    bf16, 2^-8), each p moves by at most e^(2 dz) - 1, o is rounded once."""
    o, lse, zmag, mag = ref
    fin = torch.isfinite(lse)
    assert torch.equal(torch.isfinite(got_lse), fin)
    assert bool((got_lse[~fin] == -np.inf).all()) and bool((got_o[~fin] == 0).all())
    if not bool(fin.any()):
        return
    dz = zmag * ((2.0 ** -11 if fmt == "fp8" else 0.0) + 576 * 2.0 ** -24) + 2.0 ** -20
    err = (got_lse.double() - lse).abs()[fin]
    assert bool((err <= dz[fin] + 2.0 ** -22 * lse.abs()[fin]).all()), float((err - dz[fin]).max())
    step = 2.0 ** -8 if got_o.dtype == BF else 2.0 ** -11
    p_step = 2.0 ** -8 if fmt == "bf16" else 2.0 ** -11
    bound = mag * (p_step + 2.0 ** -11 + torch.expm1(2 * dz)[..., None]) * 1.01 + step * o.abs() + 2.0 ** -24
    oerr = (got_o.double() - o).abs()
    assert bool((oerr <= bound)[fin].all()), float((oerr / bound)[fin].max())
    # the roundings are independent: in the 2-norm each leaves about a third of
    # its half step (1/sqrt 3), all of them together less than twice the largest
    rel = float((oerr[fin].square().sum() / o[fin].square().sum()).sqrt())
    assert rel <= 2 * max(step, p_step), rel


def tables(lens, page, seed, spare=1, extra_pages=2):
    need = [-(-max(int(n), 0) // page) for n in lens]
    width, total = max(max(need), 1) + spare, sum(need) + extra_pages
    order = torch.randperm(total, generator=gen(seed), device=DEV).int()
    bt = torch.zeros(len(lens), width, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        bt[b, :n] = order[at:at + n]
        at += n
    return bt, total


def random_masks(dsa, B, T, seed):
    rng = np.random.default_rng(seed)
    parents = np.array([[rng.integers(-1, i) if i else -1 for i in range(T)] for _ in range(B)]).reshape(B, T)
    return dsa.mla_sparse.draft_tree_masks(torch.tensor(parents, device=DEV))[0]


def run_tree(dsa, oracle, fmt, q_dtype, o_dtype, T, H, lens, drafts, page=64, seed=0, q_mul=1.0, scale=SCALE):
    B = len(lens)
    bt, pages = tables(lens, page, seed)
    cache = make_cache(fmt, pages, page, seed + 1, oracle)
    q = (torch.randn(B, T, H, 576, generator=gen(seed + 2), device=DEV) * q_mul).to(q_dtype)
    mask = random_masks(dsa, B, T, seed)
    ln = torch.tensor(lens, dtype=torch.int32, device=DEV)
    dl = None if drafts is None else torch.tensor(drafts, dtype=torch.int32, device=DEV)
    o = torch.full((B, T, H, 512), 7.0, dtype=o_dtype, device=DEV)
    lse = torch.full((B, T, H), 7.0, device=DEV)
    dsa.tree_mla_decode(o, lse, q, cache, bt, ln, mask, scale, dl)
    check_tree(o, lse, tree64(q, cache, bt, lens, mask, drafts, scale), fmt)
    return q, cache, bt, ln, mask, dl, o, lse


@pytest.mark.parametrize("fmt,q_dtype,o_dtype", [("fp8", BF, BF), ("fp8", HF, HF), ("f16", HF, HF), ("f16", BF, BF),
                                                  ("bf16", BF, BF), ("bf16", BF, HF)])
@pytest.mark.parametrize("T,H,lens,drafts", [
    (1, 1, [1], None), (1, 8, [1, 2, 5], None), (4, 8, [37, 4, 5], None), (3, 5, [127, 128, 129], None),
    (7, 16, [255, 256, 257], [7, 3, 1]), (2, 64, [511, 512, 513, 600], None), (64, 3, [64, 65, 190], [64, 60, 1]),
    (5, 13, [0, 1, 3, 40], [5, 5, 5, 0]), (2, 128, [70, 1030], [2, 9]), (16, 8, [1000, 33, 2049], [16, -4, 9]),
])
def test_tree_matches_64_bits(dsa, oracle, fmt, q_dtype, o_dtype, T, H, lens, drafts):
    run_tree(dsa, oracle, fmt, q_dtype, o_dtype, T, H, lens, drafts, seed=T * 7 + H)


@pytest.mark.parametrize("fmt", ["fp8", "bf16"])
@pytest.mark.parametrize("page", [1, 16, 48, 256])
def test_tree_page_sizes(dsa, oracle, fmt, page):
    run_tree(dsa, oracle, fmt, BF, BF, 6, 8, [300, 47, 49, 700], [6, 2, 6, 5], page=page, seed=page)


def test_tree_many_requests_and_long_context(dsa, oracle):
    """More row tiles than CTAs, and one request over many key slices."""
    run_tree(dsa, oracle, "fp8", BF, BF, 3, 64, [5 + 13 * b for b in range(90)], None, seed=3)
    run_tree(dsa, oracle, "fp8", BF, BF, 4, 32, [20011], None, seed=4)
    run_tree(dsa, oracle, "f16", HF, HF, 2, 8, [9973, 1, 5000], None, seed=5)


@pytest.mark.parametrize("mul", [2.0 ** 40, 2.0 ** -60])
def test_tree_bf16_q_outside_fp16_range(dsa, oracle, mul):
    """bf16 q of any magnitude; the scale undoes it, so the scores stay."""
    run_tree(dsa, oracle, "fp8", BF, BF, 3, 8, [700, 60], None, seed=6, q_mul=mul, scale=SCALE / mul)


@pytest.mark.parametrize("scale", [0.0, -SCALE, 1e-30])
def test_tree_other_scales(dsa, oracle, scale):
    """A scale of zero weighs all seen positions alike; a negative one turns the scores."""
    run_tree(dsa, oracle, "fp8", BF, BF, 3, 8, [300, 3, 700], [3, 2, 1], seed=8, scale=scale)
    run_tree(dsa, oracle, "bf16", BF, BF, 3, 8, [300, 3], None, seed=8, scale=scale)


def test_tree_rows_of_very_different_magnitude(dsa, oracle):
    """Each row of q has its own exponent range."""
    bt, pages = tables([300], 64, 1)
    cache = make_cache("fp8", pages, 64, 2, oracle)
    q = torch.randn(1, 2, 4, 576, generator=gen(3), device=DEV)
    q = (q * torch.tensor([1.0, 1e-30, 1e-3, 1e-12], device=DEV)[None, None, :, None]).to(BF)
    mask = random_masks(dsa, 1, 2, 0)
    o = torch.empty(1, 2, 4, 512, dtype=BF, device=DEV)
    lse = torch.empty(1, 2, 4, device=DEV)
    lens = torch.tensor([300], dtype=torch.int32, device=DEV)
    dsa.tree_mla_decode(o, lse, q, cache, bt, lens, mask, SCALE)
    check_tree(o, lse, tree64(q, cache, bt, [300], mask, None, SCALE), "fp8")


@pytest.mark.parametrize("fmt", ["fp8", "f16"])
def test_tree_growing_scores(dsa, oracle, fmt):
    """Scores that grow along the context move the running maximum again and again."""
    L, T, H = 1500, 2, 8
    bt, pages = tables([L], 64, 1)
    cache = make_cache(fmt, pages, 64, 2, oracle)
    q = torch.randn(1, T, H, 576, generator=gen(3), device=DEV).to(BF if fmt == "fp8" else HF)
    rows = values64(cache)
    grow = torch.linspace(0.1, 6.0, L, device=DEV)
    pos = torch.arange(L, device=DEV)
    phys = bt[0].long()[pos // 64] * 64 + pos % 64
    if fmt == "fp8":
        flat = cache.view(-1, 656)
        sc = flat[phys, 512:528].contiguous().view(F32) * grow[:, None]
        flat[phys, 512:528] = sc.contiguous().view(torch.uint8)
    else:
        cache.view(-1, 576)[phys] = (rows[phys] * grow[:, None]).to(HF)
    mask = random_masks(dsa, 1, T, 0)
    o = torch.empty(1, T, H, 512, dtype=q.dtype, device=DEV)
    lse = torch.empty(1, T, H, device=DEV)
    lens = torch.tensor([L], dtype=torch.int32, device=DEV)
    dsa.tree_mla_decode(o, lse, q, cache, bt, lens, mask, SCALE)
    check_tree(o, lse, tree64(q, cache, bt, [L], mask, None, SCALE), fmt)


def test_tree_rows_that_see_nothing(dsa, oracle):
    """Empty masks without a context give o = 0, lse = -inf; with one, the context alone."""
    T, H = 5, 8
    for lens in ([5], [25]):
        bt, pages = tables(lens, 64, 1)
        cache = make_cache("fp8", pages, 64, 2, oracle)
        q = torch.randn(1, T, H, 576, generator=gen(3), device=DEV).to(BF)
        mask = torch.tensor([[1, 0, 4, 0, -1]], dtype=torch.int64, device=DEV)
        o = torch.full((1, T, H, 512), 7.0, dtype=BF, device=DEV)
        lse = torch.full((1, T, H), 7.0, device=DEV)
        dsa.tree_mla_decode(o, lse, q, cache, bt, torch.tensor(lens, dtype=torch.int32, device=DEV), mask, SCALE)
        check_tree(o, lse, tree64(q, cache, bt, lens, mask, None, SCALE), "fp8")
        if lens == [5]:
            assert bool((lse[0, 1] == -np.inf).all()) and bool((o[0, 3] == 0).all())


@pytest.mark.parametrize("fmt", ["fp8", "f16", "bf16"])
def test_tree_never_reads_hidden_positions(dsa, oracle, fmt):
    """NaN and infinities past the sequence, in pages of no request and in a
    draft that no row sees change nothing; the table may hold anything there."""
    T, H, L = 4, 8, 150
    bt, pages = tables([L], 64, 1)
    cache = make_cache(fmt, pages, 64, 2, oracle)
    q = torch.randn(1, T, H, 576, generator=gen(3), device=DEV).to(BF)
    mask = torch.tensor([[1, 1 | 2, 0, 1 | 8]], dtype=torch.int64, device=DEV)  # draft 2 is seen by nobody
    lens = torch.tensor([L], dtype=torch.int32, device=DEV)
    keep = torch.zeros(pages * 64, dtype=torch.bool, device=DEV)
    pos = torch.arange(L, device=DEV)
    pos = pos[pos != L - T + 2]
    keep[bt[0].long()[pos // 64] * 64 + pos % 64] = True
    outs = []
    for poison in (False, True):
        c = cache.clone()
        if poison:
            flat = c.view(-1, c.shape[-1])
            bad = ~keep
            if fmt == "fp8":
                flat[bad] = 0xFF  # NaN codes, NaN scales, NaN halves
            else:
                flat[bad] = float("nan")
                flat[bad, ::3] = float("inf")
            bt = bt.clone()
            bt[0, 3:] = 2 ** 31 - 1
        o = torch.empty(1, T, H, 512, dtype=BF, device=DEV)
        lse = torch.empty(1, T, H, device=DEV)
        dsa.tree_mla_decode(o, lse, q, c, bt, lens, mask, SCALE)
        outs.append((o, lse))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


def test_tree_bad_pages_read_as_zeros(dsa, oracle):
    """Block-table entries outside the cache, and positions past the table: zero rows, counted."""
    T, H = 2, 8
    bt, pages = tables([400, 300], 64, 1, spare=0)
    cache = make_cache("fp8", pages, 64, 2, oracle)
    bt[0, 1] = -3
    bt[0, 4] = 2 ** 31 - 1
    bt[1, 0] = pages
    bt = bt[:, :6].contiguous()  # positions from 384 on are past the table
    q = torch.randn(2, T, H, 576, generator=gen(3), device=DEV).to(BF)
    mask = random_masks(dsa, 2, T, 0)
    lens = torch.tensor([400, 300], dtype=torch.int32, device=DEV)
    o = torch.empty(2, T, H, 512, dtype=BF, device=DEV)
    lse = torch.empty(2, T, H, device=DEV)
    dsa.tree_mla_decode(o, lse, q, cache, bt, lens, mask, SCALE)
    check_tree(o, lse, tree64(q, cache, bt, [400, 300], mask, None, SCALE), "fp8")


def test_tree_cache_beyond_32_bit_offsets(dsa, oracle):
    """Rows more than 2^32 bytes into the cache."""
    pages = 110_000  # 4.6 GB of 656-byte rows
    cache = torch.zeros(pages, 64, 656, dtype=torch.uint8, device=DEV)
    small = make_cache("fp8", 6, 64, 2, oracle)
    at = torch.tensor([3, 109_990, 105_000, 109_999, 60_000, 109_998], device=DEV)
    cache[at] = small
    bt = at.int()[None].contiguous()
    L, T, H = 360, 3, 8
    q = torch.randn(1, T, H, 576, generator=gen(3), device=DEV).to(BF)
    mask = random_masks(dsa, 1, T, 0)
    lens = torch.tensor([L], dtype=torch.int32, device=DEV)
    o = torch.empty(1, T, H, 512, dtype=BF, device=DEV)
    lse = torch.empty(1, T, H, device=DEV)
    dsa.tree_mla_decode(o, lse, q, cache, bt, lens, mask, SCALE)
    near = torch.arange(6, dtype=torch.int32, device=DEV)[None].contiguous()
    check_tree(o, lse, tree64(q, small, near, [L], mask, None, SCALE), "fp8")
    out = torch.empty(L, 576, dtype=BF, device=DEV)
    dsa.gather_cache(out, cache, bt, torch.tensor([0, L], dtype=torch.int32, device=DEV))
    want = torch.empty_like(out)
    dsa.gather_cache(want, small, near, torch.tensor([0, L], dtype=torch.int32, device=DEV))
    assert torch.equal(out, want)


def test_tree_strided_tables_and_repeatability(dsa, oracle):
    q, cache, bt, ln, mask, dl, o, lse = run_tree(dsa, oracle, "fp8", BF, BF, 5, 16, [900, 130, 64], [5, 2, 4], seed=9)
    wide = torch.full((3, bt.shape[1] + 9), 2 ** 30, dtype=torch.int32, device=DEV)
    wide[:, 2:2 + bt.shape[1]] = bt
    wmask = torch.full((3, 11), -1, dtype=torch.int64, device=DEV)
    wmask[:, 3:8] = mask
    wl = torch.zeros(6, dtype=torch.int32, device=DEV)
    wl[::2] = ln
    for _ in range(2):
        o2, lse2 = torch.empty_like(o), torch.empty_like(lse)
        dsa.tree_mla_decode(o2, lse2, q, cache, wide[:, 2:2 + bt.shape[1]], wl[::2], wmask[:, 3:8], SCALE, dl)
        assert torch.equal(o2, o) and torch.equal(lse2, lse)
    o3, lse3 = dsa.mla_sparse.forward_mqa_tree(q.view(15, 16, 576), cache, bt, ln, mask, SCALE, draft_lens=dl)
    assert o3.shape == (15, 16, 512) and torch.equal(o3.view_as(o), o) and torch.equal(lse3.view_as(lse), lse)


def test_tree_side_stream_and_overlapping_calls(dsa, oracle):
    """Two calls at once on two streams, each behind its own inputs' producer."""
    a = run_tree(dsa, oracle, "fp8", BF, BF, 8, 16, [3000, 500], None, seed=11)
    b = run_tree(dsa, oracle, "fp8", BF, BF, 8, 16, [2500, 700], None, seed=12)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for st, (q, cache, bt, ln, mask, dl, o, lse) in zip(streams, (a, b)):
        with torch.cuda.stream(st):
            got = [dsa.mla_sparse.forward_mqa_tree(q.clone(), cache, bt, ln, mask, SCALE) for _ in range(4)]
        outs.append(got)
    torch.cuda.synchronize()
    for got, (_, _, _, _, _, _, o, lse) in zip(outs, (a, b)):
        for o2, lse2 in got:
            assert torch.equal(o2, o) and torch.equal(lse2, lse)


def test_tree_in_a_graph_with_new_lengths(dsa, oracle):
    """One captured call serves other lengths, masks and tables of the same shapes."""
    q, cache, bt, ln, mask, dl, _, _ = run_tree(dsa, oracle, "fp8", BF, BF, 4, 16, [1500, 300], [4, 4], seed=13)
    o, lse = torch.empty(2, 4, 16, 512, dtype=BF, device=DEV), torch.empty(2, 4, 16, device=DEV)
    dsa.tree_mla_decode(o, lse, q, cache, bt, ln, mask, SCALE, dl)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dsa.tree_mla_decode(o, lse, q, cache, bt, ln, mask, SCALE, dl)
    for lens, drafts in (([1500, 300], [4, 4]), ([7, 299], [2, 4]), ([1400, 0], [1, 4])):
        ln.copy_(torch.tensor(lens, dtype=torch.int32))
        dl.copy_(torch.tensor(drafts, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        check_tree(o, lse, tree64(q, cache, bt, lens, mask, drafts, SCALE), "fp8")


def test_tree_of_a_line_equals_the_spec_rows(dsa, oracle):
    """A line of drafts over a context below the top-k: the same rows as the
    sparse decode of every position (two kernels, each within its bounds)."""
    B, T, H, L = 2, 3, 64, 200
    lens = [L, L - 30]
    bt, pages = tables(lens, 64, 1)
    cache = make_cache("fp8", pages, 64, 2, oracle)
    q = torch.randn(B, T, H, 576, generator=gen(3), device=DEV).to(BF)
    ln = torch.tensor(lens, dtype=torch.int32, device=DEV)
    mask = dsa.mla_sparse.draft_tree_masks(torch.arange(T, device=DEV)[None].expand(B, -1) - 1)[0]
    o, lse = dsa.mla_sparse.forward_mqa_tree(q, cache, bt, ln, mask, SCALE)
    idx = torch.arange(256, dtype=torch.int32, device=DEV).expand(B * T, -1).contiguous()
    o2, lse2 = dsa.mla_sparse.forward_mqa_sparse(q.view(B * T, H, 576), cache, idx, 256, bt, ln, SCALE)
    ref = tree64(q, cache, bt, lens, mask, None, SCALE)
    check_tree(o, lse, ref, "fp8")
    assert float((lse.view(-1, H) - lse2).abs().max()) <= 2e-3  # the decode's own lse tolerance
    rel = float((o.view(-1, H, 512).double() - o2.double()).norm() / o2.double().norm())
    assert rel <= 2 * 2.0 ** -8  # each within half a bf16 step and smaller roundings of the same values


def test_tree_refusals(dsa, oracle):
    q, cache, bt, ln, mask, dl, o, lse = run_tree(dsa, oracle, "fp8", BF, BF, 2, 8, [40], [2], seed=1)

    def call(**k):
        a = dict(o=o, lse=lse, q=q, kv_cache=cache, block_table=bt, seq_lens=ln, tree_mask=mask, scale=SCALE, draft_lens=dl)
        a.update(k)
        dsa.tree_mla_decode(**a)

    for bad in [dict(q=q.float()), dict(q=q[..., :512]), dict(o=o[..., :256]), dict(lse=lse.half()), dict(lse=lse[:, :1]),
                dict(kv_cache=cache[..., :640]), dict(kv_cache=cache.transpose(0, 1)), dict(block_table=bt.long()),
                dict(block_table=bt.cpu()), dict(seq_lens=ln.cpu()), dict(seq_lens=ln.long()), dict(tree_mask=mask.int()),
                dict(tree_mask=mask[:, :1]), dict(tree_mask=mask.cpu()), dict(draft_lens=dl.long()), dict(draft_lens=dl.cpu()),
                dict(block_table=bt[:0]), dict(seq_lens=ln[:0]), dict(draft_lens=dl[:0]),
                dict(q=q.half(), kv_cache=make_cache("bf16", 3, 64, 1, oracle))]:
        with pytest.raises(RuntimeError):
            call(**bad)
    # an empty batch is no work
    e = dict(q=q[:0], o=o[:0], lse=lse[:0], tree_mask=mask[:0])
    call(**e)


# ------------------------------------------------------------------- rotary
def rope_f32(x, cos_sin, pos, off, neox):
    """f32, each product and sum rounded, then one rounding to x's type."""
    r = cos_sin.shape[1]
    p = pos.clamp(0, cos_sin.shape[0] - 1)
    c, s = cos_sin[p][:, None, :r // 2], cos_sin[p][:, None, r // 2:]
    out = x.clone()
    part = x[..., off:off + r].float()
    a, b = (part[..., :r // 2], part[..., r // 2:]) if neox else (part[..., 0::2], part[..., 1::2])
    ac, bs, bc, as_ = a * c, b * s, b * c, a * s
    o1, o2 = (ac - bs).to(x.dtype), (bc + as_).to(x.dtype)
    if neox:
        out[..., off:off + r // 2], out[..., off + r // 2:off + r] = o1, o2
    else:
        out[..., off:off + r:2], out[..., off + 1:off + r:2] = o1, o2
    return out


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("T,H,W,r,off,lead_in,lead_out", [
    (1, 1, 64, 64, 0, 0, 0), (5, 64, 64, 64, 0, 192, 512), (3, 7, 200, 96, 40, 0, 8), (33, 2, 66, 32, 1, 0, 0),
    (4, 3, 130, 6, 3, 1, 5), (1000, 16, 128, 64, 64, 0, 0), (2, 128, 576, 64, 512, 0, 0), (7, 1, 2, 2, 0, 0, 0),
    (300, 5, 72, 64, 8, 4, 4), (3, 1, 2048, 2048, 0, 0, 0),
])
def test_rotary_matches_f32_bit_for_bit(dsa, dtype, neox, T, H, W, r, off, lead_in, lead_out):
    g = gen(T + W)
    x = torch.randn(T, H, lead_in + W, generator=g, device=DEV).to(dtype)[..., lead_in:]
    buf = torch.full((T, H, lead_out + W + 3), 5.0, dtype=dtype, device=DEV)
    out = buf[..., lead_out:lead_out + W]
    table = dsa.rope.rope_cos_sin_cache(r, 5000, device=DEV)
    pos = torch.randint(0, 5000, (T,), generator=g, device=DEV)
    pos[0], pos[-1] = 4999 if T > 1 else 0, -3  # out of the table: clamped
    dsa.rotary_embedding(out, x, pos, table, neox, off)
    want = rope_f32(x, table, pos, off, neox)
    assert torch.equal(out, want)
    assert bool((buf[..., :lead_out] == 5).all()) and bool((buf[..., lead_out + W:] == 5).all())
    same = x.clone()
    dsa.rotary_embedding(same, same, pos, table, neox, off)
    assert torch.equal(same, want)


def test_rotary_against_64_bits_and_back(dsa):
    """Half a step per rounding of the formula in 64 bits; minus the angle undoes it."""
    T, H, r = 64, 4, 64
    x = torch.randn(T, H, r, generator=gen(1), device=DEV)
    table = dsa.rope.rope_cos_sin_cache(r, 200_000, scaling={"type": "yarn", "factor": 40.0, "original_max_position": 4096,
                                                             "mscale": 1.0, "mscale_all_dim": 1.0}, device=DEV)
    pos = torch.randint(0, 200_000, (T,), generator=gen(2), device=DEV)
    out = torch.empty_like(x)
    dsa.rotary_embedding(out, x, pos, table, True)
    c, s = table.double()[pos][:, None, :32], table.double()[pos][:, None, 32:]
    a, b = x.double()[..., :32], x.double()[..., 32:]
    want = torch.cat([a * c - b * s, b * c + a * s], -1)
    size = torch.cat([(a * c).abs() + (b * s).abs()] * 1 + [(b * c).abs() + (a * s).abs()], -1)
    assert bool(((out.double() - want).abs() <= 2.0 ** -24 * (size + want.abs()) * 1.0001).all())
    back = table.clone()
    back[:, 32:] *= -1
    again = torch.empty_like(x)
    dsa.rotary_embedding(again, out, pos, back, True)
    # two rotations, three roundings each, and cos^2 + sin^2 of rounded entries within 2^-23 of 1
    assert float((again - x).abs().max()) <= 8 * 2.0 ** -24 * float(x.abs().max()) * 2


def test_rotary_broadcast_heads_streams_and_refusals(dsa):
    table = dsa.rope.rope_cos_sin_cache(64, 100, device=DEV)
    x = torch.randn(6, 1, 64, generator=gen(1), device=DEV).to(BF)
    pos = torch.arange(6, device=DEV)
    out = torch.empty(6, 5, 64, dtype=BF, device=DEV)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        dsa.rotary_embedding(out, x.expand(6, 5, 64), pos, table)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(out, rope_f32(x, table, pos, 0, False).expand(6, 5, 64))
    dsa.rotary_embedding(out[:0], x[:0].expand(0, 5, 64), pos[:0], table)
    for bad in [dict(x=x.int()), dict(x=x.half()), dict(positions=pos.int()), dict(positions=pos[:5]),
                dict(positions=pos.cpu()), dict(cos_sin_cache=table.half()), dict(cos_sin_cache=table[:0]),
                dict(cos_sin_cache=table.cpu()), dict(rope_offset=2), dict(rope_offset=-1),
                dict(out=out.transpose(0, 1)), dict(cos_sin_cache=dsa.rope.rope_cos_sin_cache(128, 10, device=DEV))]:
        a = dict(out=out, x=x.expand(6, 5, 64), positions=pos, cos_sin_cache=table, is_neox=False, rope_offset=0)
        a.update(bad)
        with pytest.raises(RuntimeError):
            dsa.rotary_embedding(**a)


# ------------------------------------------------------------------- gather
def plain_rows(cache, out_dtype):
    rows = cache.reshape(-1, cache.shape[-1])
    if cache.dtype != torch.uint8:
        return rows.float().to(out_dtype)
    groups = 4 if rows.shape[1] == 656 else 1
    code = rows[:, :128 * groups].contiguous().view(torch.float8_e4m3fn).float().view(-1, groups, 128)
    scale = rows[:, 128 * groups:132 * groups].contiguous().view(F32)
    v = (code * scale[..., None]).flatten(1)
    if groups == 4:
        v = torch.cat([v, rows[:, 528:].contiguous().view(HF).float()], 1)
    return v.to(out_dtype)


def idxk_cache(pages, page, seed):
    x = torch.randn(pages * page, 128, generator=gen(seed), device=DEV)
    s = x.abs().amax(1, keepdim=True) / 448.0
    raw = torch.empty(pages * page, 132, dtype=torch.uint8, device=DEV)
    raw[:, :128] = (x / s).to(torch.float8_e4m3fn).view(torch.uint8)
    raw[:, 128:] = s.view(torch.uint8)
    return raw.view(pages, page, 132)


@pytest.mark.parametrize("fmt", ["fp8", "idxk", "f16", "bf16", "f16w128"])
@pytest.mark.parametrize("out_dtype", [BF, HF])
@pytest.mark.parametrize("lens,starts,page", [([1], None, 64), ([0, 5, 0, 200, 1], None, 64), ([64, 65, 63], [3, 0, 100], 64),
                                              ([700], [130], 16), ([33, 40], [7, 1], 5)])
def test_gather_bit_exact(dsa, oracle, fmt, out_dtype, lens, starts, page):
    ends = [n + (0 if starts is None else starts[b]) for b, n in enumerate(lens)]
    bt, pages = tables(ends, page, 1)
    cache = (idxk_cache(pages, page, 2) if fmt == "idxk" else
             make_cache("f16", pages, page, 2, oracle)[..., :128].contiguous() if fmt == "f16w128" else
             make_cache(fmt, pages, page, 2, oracle))
    cu = torch.tensor([0] + lens, dtype=torch.int32, device=DEV).cumsum(0).int()
    n = int(cu[-1])
    want_rows = plain_rows(cache, out_dtype)
    buf = torch.full((n + 3, want_rows.shape[1] + 16), 9.0, dtype=out_dtype, device=DEV)
    out = buf[:, 8:8 + want_rows.shape[1]]
    st = None if starts is None else torch.tensor(starts, dtype=torch.int32, device=DEV)
    dsa.gather_cache(out, cache, bt, cu, st)
    at = 0
    for b, k in enumerate(lens):
        pos = torch.arange(k, device=DEV) + (0 if starts is None else starts[b])
        rows = bt[b].long()[pos // page] * page + pos % page
        assert torch.equal(out[at:at + k], want_rows[rows]), b
        at += k
    assert bool((out[n:] == 9).all()) and bool((buf[:, :8] == 9).all())  # rows behind the last request


def test_gather_bad_pages_short_outputs_and_refusals(dsa, oracle):
    cache = make_cache("fp8", 4, 64, 2, oracle)
    bt = torch.tensor([[1, -1, 3], [4, 2 ** 31 - 1, 0]], dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 200, 300], dtype=torch.int32, device=DEV)
    out = torch.full((300, 576), 9.0, dtype=BF, device=DEV)
    dsa.gather_cache(out, cache, bt, cu)
    rows = plain_rows(cache, BF)
    assert torch.equal(out[:64], rows[64:128]) and bool((out[64:128] == 0).all()) and torch.equal(out[128:192], rows[192:])
    assert bool((out[192:300] == 0).all())  # past the table, pages outside the cache
    part = torch.full((70, 576), 9.0, dtype=BF, device=DEV)
    dsa.gather_cache(part, cache, bt, cu)  # out shorter than the requests: its rows only
    assert torch.equal(part, out[:70])
    neg = torch.tensor([-5, 0], dtype=torch.int32, device=DEV)
    dsa.gather_cache(part, cache, bt, cu, neg)
    assert bool((part[:5] == 0).all()) and torch.equal(part[5:69], rows[64:128])
    one = torch.empty(1, 576, dtype=HF, device=DEV)
    dsa.gather_cache(one, cache, bt, cu)
    assert torch.equal(one, plain_rows(cache, HF)[64:65])
    for bad in [dict(out=out.float()), dict(out=out[:, :512]), dict(cache=cache[..., :640]), dict(cache=cache.transpose(0, 1)),
                dict(block_table=bt.long()), dict(block_table=bt.cpu()), dict(block_table=bt[:1]), dict(cu_seq_lens=cu.long()),
                dict(cu_seq_lens=cu.cpu()), dict(cu_seq_lens=cu[:0]), dict(seq_starts=neg.long()), dict(seq_starts=neg[:1]),
                dict(out=torch.empty(9, 580, dtype=BF, device=DEV)[:, 2:578])]:
        a = dict(out=out, cache=cache, block_table=bt, cu_seq_lens=cu, seq_starts=None)
        a.update(bad)
        with pytest.raises(RuntimeError):
            dsa.gather_cache(**a)
    dsa.gather_cache(out[:0], cache, bt, cu)


def test_gather_reads_what_the_writers_wrote(dsa):
    """Written, quantised and read back: half an e4m3 step of each value (2^-4
    of it, or of the smallest normal code's scale below that) and bf16's."""
    n, page = 100, 64
    kv_c = torch.randn(n, 512, generator=gen(1), device=DEV).to(BF)
    k_pe = torch.randn(n, 64, generator=gen(2), device=DEV).to(BF)
    cache = torch.zeros(3, page, 656, dtype=torch.uint8, device=DEV)
    bt = torch.tensor([[2, 0]], dtype=torch.int32, device=DEV)
    pos = torch.arange(n, device=DEV)
    slots = (bt[0].long()[pos // page] * page + pos % page).int()
    dsa.ops.concat_and_cache_mla(kv_c, k_pe, cache, slots)
    out = torch.empty(n, 576, dtype=BF, device=DEV)
    dsa.gather_cache(out, cache, bt, torch.tensor([0, n], dtype=torch.int32, device=DEV))
    v = kv_c.double()
    scale = v.view(n, 4, 128).abs().amax(2, keepdim=True).expand(-1, -1, 128).reshape(n, 512) / 448.0
    bound = torch.maximum(v.abs() * 2.0 ** -4, scale * 2.0 ** -10) * 1.0001
    assert bool(((out[:, :512].double() - v).abs() <= bound * (1 + 2.0 ** -8) + v.abs() * 2.0 ** -8).all())
    assert torch.equal(out[:, 512:], k_pe.half().float().to(BF))


# ------------------------------------------------------------------- commit
@pytest.mark.parametrize("row,dtype", [(656, torch.uint8), (132, torch.uint8), (576, BF), (128, HF)])
@pytest.mark.parametrize("layers", [1, 3, 130])
def test_commit_moves_rows(dsa, row, dtype, layers):
    page, T = 16, 64
    lens, drafts = [100, 64, 70, 5, 90], [64, 64, 12, 5, 0]
    bt, pages = tables(lens, page, 1)
    pool = torch.randint(0, 255, (layers, pages, page, row), generator=gen(2), device=DEV, dtype=torch.int32).to(dtype)
    rng = np.random.default_rng(3)
    acc = np.full((5, 40), -1, np.int32)
    acc[0, :40] = np.sort(rng.permutation(64)[:40])        # long path: most moves overlap
    acc[1, :3] = [0, 1, 2]                                 # already in place
    acc[2, :6] = [3, 3, 1, 0, 11, 12]                      # the same row twice, backwards, 12: no draft
    acc[3, :5] = [4, -7, 2, 99, 0]
    acc[4, :2] = [0, 1]                                    # no drafts
    want = pool.clone()
    flat, wflat = pool.view(layers, -1, row), want.view(layers, -1, row)

    def at(b, p):
        return int(bt[b, p // page]) * page + p % page

    for b in range(5):
        pre = lens[b] - drafts[b]
        for k, a in enumerate(acc[b]):
            if 0 <= a < drafts[b] and k < drafts[b]:
                wflat[:, at(b, pre + k)] = flat[:, at(b, pre + int(a))]
    args = (bt, torch.tensor(lens, dtype=torch.int32, device=DEV), torch.tensor(acc, device=DEV),
            torch.tensor(drafts, dtype=torch.int32, device=DEV))
    dsa.commit_draft_rows(list(pool.unbind(0)), *args)
    assert torch.equal(pool, want)


def test_commit_bad_pages_and_refusals(dsa):
    cache = torch.arange(4 * 16 * 132, device=DEV).to(torch.uint8).view(4, 16, 132)
    bt = torch.tensor([[-1, 2, 9]], dtype=torch.int32, device=DEV)
    ln, dl = torch.tensor([40], dtype=torch.int32, device=DEV), torch.tensor([40], dtype=torch.int32, device=DEV)
    before = cache.clone()
    acc = torch.full((1, 30), -1, dtype=torch.int32, device=DEV)
    acc[0, 0], acc[0, 17], acc[0, 18] = 20, 3, 35  # into a bad page, from one, from another
    dsa.commit_draft_rows([cache], bt, ln, acc, dl)
    assert torch.equal(cache, before)
    acc[0, 16] = 20
    dsa.commit_draft_rows([cache], bt, ln, acc, dl)
    before[2, 0] = before[2, 4]
    assert torch.equal(cache, before)
    for bad in [dict(caches=[cache, cache]), dict(caches=[cache, cache[:2]]), dict(caches=[cache.transpose(0, 1)]),
                dict(block_table=bt.long()), dict(accepted=acc.long()), dict(accepted=acc.cpu()), dict(seq_lens=ln.cpu()),
                dict(draft_lens=dl.cpu()), dict(draft_lens=dl[:0]), dict(accepted=acc[0]),
                dict(accepted=torch.zeros(1, 65, dtype=torch.int32, device=DEV)),
                dict(caches=[torch.zeros(2, 4, 130, dtype=torch.uint8, device=DEV)])]:
        a = dict(caches=[cache], block_table=bt, seq_lens=ln, accepted=acc, draft_lens=dl)
        a.update(bad)
        with pytest.raises(RuntimeError):
            dsa.commit_draft_rows(**a)
    dsa.commit_draft_rows([], bt, ln, acc, dl)


# ---------------------------------------------------------- all of them together
def test_verify_a_tree_end_to_end(dsa):
    """rotary -> write -> tree attention -> commit: the accepted path's rows
    attend and end up in the cache as if it had been decoded as a line."""
    H, page, L, T = 8, 64, 200, 6
    parents = torch.tensor([[-1, -1, 0, 1, 1, 3]], device=DEV)
    path = [1, 3, 5]
    mask, depth = dsa.mla_sparse.draft_tree_masks(parents)
    table = dsa.rope.rope_cos_sin_cache(64, 1024, device=DEV)
    g = gen(4)
    ctx_c, ctx_pe = torch.randn(L, 512, generator=g, device=DEV).to(BF), torch.randn(L, 64, generator=g, device=DEV).to(BF)
    new_c, new_pe = torch.randn(T, 512, generator=g, device=DEV).to(BF), torch.randn(T, 64, generator=g, device=DEV).to(BF)
    nope, q_pe = torch.randn(T, H, 512, generator=g, device=DEV).to(BF), torch.randn(T, H, 64, generator=g, device=DEV).to(BF)
    bt = torch.tensor([[2, 0, 3, 1]], dtype=torch.int32, device=DEV)

    def slots(p):
        return (bt[0].long()[p // page] * page + p % page).int()

    def query(rows, pos):
        q = torch.empty(len(rows), H, 576, dtype=BF, device=DEV)
        q[..., :512] = nope[rows]
        dsa.rotary_embedding(q[..., 512:], q_pe[rows], pos, table)
        return q

    def fresh():
        c = torch.zeros(4, page, 656, dtype=torch.uint8, device=DEV)
        p = torch.arange(L, device=DEV)
        dsa.ops.concat_and_cache_mla(ctx_c, ctx_pe, c, slots(p), positions=p, cos_sin_cache=table)
        return c

    tree = fresh()
    at = L + torch.arange(T, device=DEV)
    pos = L + depth[0]
    dsa.ops.concat_and_cache_mla(new_c, new_pe, tree, slots(at), positions=pos, cos_sin_cache=table)
    n = torch.tensor([L + T], dtype=torch.int32, device=DEV)
    o, lse = dsa.mla_sparse.forward_mqa_tree(query(list(range(T)), pos), tree, bt, n, mask, SCALE)
    dsa.commit_draft_rows([tree], bt, n, torch.tensor([path], dtype=torch.int32, device=DEV),
                          torch.tensor([T], dtype=torch.int32, device=DEV))
    line = fresh()
    lp = L + torch.arange(3, device=DEV)
    dsa.ops.concat_and_cache_mla(new_c[path], new_pe[path], line, slots(lp), positions=lp, cos_sin_cache=table)
    keep = slots(torch.arange(L + 3, device=DEV)).long()
    assert torch.equal(tree.view(-1, 656)[keep], line.view(-1, 656)[keep])
    chain, _ = dsa.mla_sparse.draft_tree_masks(torch.arange(3, device=DEV)[None] - 1)
    o2, lse2 = dsa.mla_sparse.forward_mqa_tree(query(path, lp), line, bt, torch.tensor([L + 3], dtype=torch.int32, device=DEV),
                                               chain, SCALE)
    # the same keys in another order: f32 sums of 203 and 576 terms, and o's last step
    assert float((lse[path] - lse2).abs().max()) <= 1e-4
    assert bool(((o[path].double() - o2.double()).abs() <= 2.0 ** -7 * o2.double().abs() + 2.0 ** -11).all())
    back = torch.empty(L + 3, 576, dtype=BF, device=DEV)
    dsa.gather_cache(back, tree, bt, torch.tensor([0, L + 3], dtype=torch.int32, device=DEV))
    ctx = torch.empty(L + 3, 1, 64, dtype=BF, device=DEV)
    both = torch.cat([ctx_pe, new_pe[path]])[:, None]
    dsa.rotary_embedding(ctx, both, torch.arange(L + 3, device=DEV), table)
    # the writer rounds the rotated key to fp16, the operator to bf16
    assert bool(((back[:, 512:].double() - ctx[:, 0].double()).abs() <= 2.0 ** -7 * ctx[:, 0].double().abs() + 2.0 ** -20).all())


def test_tree_lengths_of_every_kind_in_one_batch(dsa, oracle):
    """Requests whose scores take one, two or two finer products follow one
    another in a pair's run, with rows of empty requests between them."""
    lens = [1000, 20000, 40000, 3, 1024, 1025, 0, 32768, 32769, 1, 700]
    run_tree(dsa, oracle, "fp8", BF, BF, 2, 8, lens, None, seed=21)
    run_tree(dsa, oracle, "fp8", HF, HF, 3, 64, lens[::-1], [3, 1, 2, 3, 0, 3, 3, 3, 2, 3, 3], seed=22)


@pytest.mark.parametrize("lens", [[1, 2, 5, 40], [130, 600, 1024], [1025, 1500, 3001], [9000, 17001]])
def test_tree_scores_keep_the_scale(dsa, oracle, lens):
    """Up to 32768 positions an fp8 key enters the scores with 2^-16 of its value:
    the scale's second part has 2^-6 of it and is rounded to f16, as its product
    with the code is (2^-17 each). The errors are independent, so lse's, which
    averages scores', has no larger deviation than 2^-16 / sqrt 3 of the score's
    terms in the 2-norm; an f32 sum of the 2 * 576 terms adds sqrt(1152) 2^-24 of
    partial sums that are at most about twice that norm."""
    q, cache, bt, ln, mask, dl, o, lse = run_tree(dsa, oracle, "fp8", BF, BF, 3, 16, lens, None, seed=23)
    ref = tree64(q, cache, bt, lens, mask, None, SCALE)[1]
    fin = torch.isfinite(ref)
    k2 = values64(cache).square().mean(0)
    norm = (q.double().square() @ k2).sqrt()[fin].max() * SCALE
    rms = (lse.double() - ref)[fin].square().mean().sqrt()
    tol = (2.0 ** -16 / 3 ** 0.5 + 2 * 1152 ** 0.5 * 2.0 ** -24) * norm
    assert float(rms) <= float(tol), (float(rms), float(tol))


@pytest.mark.parametrize("lens", [[700, 3], [1500, 2100], [33000]])
def test_tree_scales_of_every_size(dsa, oracle, lens):
    """Groups' scales from 2^-24 to 2^2 side by side, and groups of scale zero; each
    element of a key is off by at most half an f16 step of itself or 2^-25."""
    bt, pages = tables(lens, 64, 31)
    cache = make_cache("fp8", pages, 64, 32, oracle)
    rows = cache.view(-1, 656)
    scale = rows[:, 512:528].contiguous().view(F32)
    power = torch.randint(-17, 2, scale.shape, generator=gen(33), device=DEV)
    power[::5] = torch.randint(-17, 10, power[::5].shape, generator=gen(34), device=DEV)
    scale = torch.ldexp(scale, power)
    scale[7::11, 1] = 0.0
    rows[:, 512:528] = scale.contiguous().view(torch.uint8)
    B, T, H = len(lens), 2, 5
    q = (torch.randn(B, T, H, 576, generator=gen(35), device=DEV) * 2.0 ** -8).to(BF)
    mask = random_masks(dsa, B, T, 36)
    ln = torch.tensor(lens, dtype=torch.int32, device=DEV)
    o, lse = torch.empty(B, T, H, 512, dtype=BF, device=DEV), torch.empty(B, T, H, device=DEV)
    dsa.tree_mla_decode(o, lse, q, cache, bt, ln, mask, SCALE)
    check_tree(o, lse, tree64(q, cache, bt, lens, mask, None, SCALE), "fp8")


def test_commit_refuses_caches_that_overlap(dsa):
    pool = torch.zeros(5, 16, 132, dtype=torch.uint8, device=DEV)
    bt = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    one = torch.ones(1, dtype=torch.int32, device=DEV)
    acc = torch.full((1, 1), -1, dtype=torch.int32, device=DEV)
    dsa.commit_draft_rows([pool[3:5], pool[0:2]], bt, one, acc, one)
    with pytest.raises(RuntimeError, match="overlap"):
        dsa.commit_draft_rows([pool[0:3], pool[4:5].expand(3, 16, 132).contiguous(), pool[1:4]], bt, one, acc, one)


def test_rotary_out_in_other_columns_of_x(dsa):
    """x and out interleaved in one buffer; in place with heads farther apart than tokens."""
    table = dsa.rope.rope_cos_sin_cache(64, 100, device=DEV)
    pos = torch.arange(7, device=DEV)
    buf = torch.randn(7, 5, 192, generator=gen(2), device=DEV).to(BF)
    want = buf.clone()
    want[..., 128:] = rope_f32(buf[..., :64].contiguous(), table, pos, 0, False)
    dsa.rotary_embedding(buf[..., 128:], buf[..., :64], pos, table)
    assert torch.equal(buf, want)
    x = torch.randn(5, 7, 64, generator=gen(3), device=DEV).to(BF)
    want = rope_f32(x.transpose(0, 1).contiguous(), table, pos, 0, True)
    dsa.rotary_embedding(x.transpose(0, 1), x.transpose(0, 1), pos, table, True)
    assert torch.equal(x.transpose(0, 1), want)


def test_commit_gather_and_rotary_in_a_graph(dsa):
    """Captured once, replayed with other lengths, paths, positions and contents."""
    B, T, page = 3, 6, 16
    cache = torch.zeros(40, page, 576, dtype=HF, device=DEV)
    bt = torch.randperm(36, generator=gen(1), device=DEV).view(B, 12).int()
    lens, drafts, cu = (torch.zeros(n, dtype=torch.int32, device=DEV) for n in (B, B, B + 1))
    acc = torch.full((B, T), -1, dtype=torch.int32, device=DEV)
    pos = torch.zeros(9, dtype=torch.int64, device=DEV)
    table = dsa.rope.rope_cos_sin_cache(64, 50, device=DEV)
    x = torch.zeros(9, 3, 64, dtype=BF, device=DEV)
    out, turned = torch.zeros(200, 576, dtype=BF, device=DEV), torch.zeros_like(x)

    def step():
        dsa.commit_draft_rows([cache], bt, lens, acc, drafts)
        dsa.gather_cache(out, cache, bt, cu)
        dsa.rotary_embedding(turned, x, pos, table)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed, (n, d) in enumerate([([30, 6, 61], [6, 3, 1]), ([0, 64, 17], [2, 6, 6]), ([1, 1, 190], [1, 0, 6])]):
        cache.copy_(torch.randn(cache.shape, generator=gen(seed), device=DEV))
        x.copy_(torch.randn(x.shape, generator=gen(seed + 9), device=DEV))
        pos.copy_(torch.randint(0, 50, pos.shape, generator=gen(seed), device=DEV))
        lens.copy_(torch.tensor(n))
        drafts.copy_(torch.tensor(d))
        cu.copy_(torch.tensor([0, *np.cumsum(np.minimum(n, 66)).tolist()]))
        acc.fill_(-1)
        want = cache.clone().view(-1, 576)
        row = lambda b, p: int(bt[b, p // page]) * page + p % page
        for b in range(B):
            path = [k for k in range(1, d[b], 2)]
            acc[b, :len(path)] = torch.tensor(path, dtype=torch.int32)
            old = want.clone()
            for k, a in enumerate(path):
                if n[b] - d[b] >= 0:
                    want[row(b, n[b] - d[b] + k)] = old[row(b, n[b] - d[b] + a)]
        out.fill_(3.0)
        graph.replay()
        assert torch.equal(cache.view(-1, 576), want)
        rows = [row(b, p) for b in range(B) for p in range(min(n[b], 66))]
        assert torch.equal(out[:len(rows)], want[rows].to(BF)) and bool((out[len(rows):] == 3.0).all())
        assert torch.equal(turned, rope_f32(x, table, pos, 0, False))


@pytest.mark.parametrize("fmt", ["fp8", "bf16"])
def test_one_tree_and_one_table_row_for_a_batch(dsa, oracle, fmt):
    """Masks, tables and paths expanded over the batch give what their copies give."""
    B, T, H, L = 5, 6, 8, 300
    row, pages = tables([L], 64, 1)
    cache = make_cache(fmt, pages, 64, 2, oracle)
    q = torch.randn(B, T, H, 576, generator=gen(3), device=DEV).to(BF)
    tree = random_masks(dsa, 1, T, 4)
    lens = [300, 299, 64, 7, 130]
    ln = torch.tensor(lens, dtype=torch.int32, device=DEV)
    outs = []
    for share in (False, True):
        mask, bt = tree.expand(B, T), row.expand(B, row.shape[1])
        if not share:
            mask, bt = mask.contiguous(), bt.contiguous()
        o, lse = torch.empty(B, T, H, 512, dtype=BF, device=DEV), torch.empty(B, T, H, device=DEV)
        dsa.tree_mla_decode(o, lse, q, cache, bt, ln, mask, SCALE)
        back = torch.full((sum(lens), 576), 9.0, dtype=BF, device=DEV)
        cu = torch.tensor([0, *np.cumsum(lens)], dtype=torch.int32, device=DEV)
        dsa.gather_cache(back, cache, bt, cu)
        outs.append((o, lse, back))
    check_tree(outs[0][0], outs[0][1], tree64(q, cache, row.expand(B, -1), lens, tree.expand(B, T), None, SCALE), fmt)
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    half = torch.as_strided(tree.expand(B, T).contiguous(), (B, T), (T - 1, 1))  # rows that overlap in part
    with pytest.raises(RuntimeError):
        dsa.tree_mla_decode(outs[0][0], outs[0][1], q, cache, row.expand(B, -1), ln, half, SCALE)


def test_commit_of_one_path_for_a_batch(dsa):
    B, T, page = 3, 8, 16
    lens = [40, 20, 33]
    bt, pages = tables(lens, page, 5)
    pool = torch.randint(0, 255, (pages, page, 132), generator=gen(6), device=DEV, dtype=torch.int32).to(torch.uint8)
    acc = torch.tensor([[1, 3, 4, 7, -1]], dtype=torch.int32, device=DEV)
    ln, dl = torch.tensor(lens, dtype=torch.int32, device=DEV), torch.full((B,), T, dtype=torch.int32, device=DEV)
    want = pool.clone()
    dsa.commit_draft_rows([want], bt, ln, acc.expand(B, -1).contiguous(), dl)
    assert not torch.equal(want, pool)
    before = pool.clone()
    with pytest.raises(RuntimeError, match="row of the block table"):
        dsa.commit_draft_rows([pool], bt[:1].expand(B, -1), ln, acc.expand(B, -1), dl)
    assert torch.equal(pool, before)
    dsa.commit_draft_rows([pool], bt, ln, acc.expand(B, -1), dl)
    assert torch.equal(pool, want)


@pytest.mark.parametrize("fmt,dtype", [("fp8", HF), ("f16", HF), ("bf16", BF)])
@pytest.mark.parametrize("at", [0, 70_000, 131_071])
def test_tree_many_faint_keys_beside_a_strong_one(dsa, oracle, fmt, dtype, at):
    """One key 17.5 nats above 131,071 others, whose weights of e^-17.5 = 1.7 * 2^-26
    add up to 0.0033 of the row. As many requests as there are CTA pairs, so that a
    pair's run is a whole context. All values are 1 but the strong key's, 1/2, so o
    = (1/2 + n w) / (1 + n w). Off are: a faint probability, by at most half a step of
    the 16-bit type (2^-11, bf16 2^-8) or 2^-25 of a scale of 2^7; its product, once the
    accumulator holds the strong one (2^6: last place 2^-17), by less than a quarter of
    that place, 2^-19 / 2^7 of o; the sum, by half a step at each of its 1024 tiles; o,
    by its own half step. (Faint probabilities that became zeros made 0.0033.)"""
    n, B, page = 131_072, torch.cuda.get_device_properties(0).multi_processor_count // 2, 64
    pages = n // page
    x = torch.zeros(n, 576, device=DEV)
    x[:, :512] = 1.0
    x[at, :512] = 0.5
    x[at, 575] = 1.0  # only the rotary part of q is set: the scores
    if fmt == "fp8":
        cache = torch.zeros(n, 656, dtype=torch.uint8, device=DEV)
        cache[:, :512] = x[:, :512].to(torch.float8_e4m3fn).view(torch.uint8)
        cache[:, 512:528] = torch.ones(n, 4, device=DEV).view(torch.uint8)
        cache[:, 528:] = x[:, 512:].half().contiguous().view(torch.uint8)
        cache = cache.view(pages, page, 656)
    else:
        cache = x.to(HF if fmt == "f16" else BF).view(pages, page, 576)
    q = torch.zeros(B, 1, 2, 576, dtype=dtype, device=DEV)
    q[..., 575] = 17.5
    bt = torch.arange(pages, dtype=torch.int32, device=DEV)[None].expand(B, -1).contiguous()
    ln = torch.full((B,), n, dtype=torch.int32, device=DEV)
    mask = torch.ones(B, 1, dtype=torch.int64, device=DEV)
    o, lse = torch.empty(B, 1, 2, 512, dtype=dtype, device=DEV), torch.empty(B, 1, 2, device=DEV)
    dsa.tree_mla_decode(o, lse, q, cache, bt, ln, mask, 1.0)
    w = (n - 1) * np.exp(-17.5)
    half = 2.0 ** -8 if dtype == BF else 2.0 ** -11
    want = (0.5 + w) / (1 + w)
    total = (n // 128 + 128) * 2.0 ** -24  # of the sum: tiles, and the additions inside one and of the quarters
    tol = w * half + n * 2.0 ** -32 + (n - at) * 2.0 ** -26 + want * total + half * want
    err = float((o.double() - want).abs().max())
    assert err <= tol, (err, tol)
    assert float((lse.double() - (17.5 + np.log1p(w))).abs().max()) <= total + 2.0 ** -20 + 2.0 ** -22 * 17.5


@pytest.mark.parametrize("fmt,served", [("fp8", HF), ("f16", HF), ("bf16", BF)])
def test_forward_mqa_tree_takes_f32_queries_and_64_bit_integers(dsa, oracle, fmt, served):
    """f32 q is rounded to the type that the cache's products take; o comes in it."""
    B, T, H, lens, drafts = 2, 3, 8, [300, 70], [3, 2]
    bt, pages = tables(lens, 64, 1)
    cache = make_cache(fmt, pages, 64, 2, oracle)
    q = torch.randn(B, T, H, 576, generator=gen(3), device=DEV)
    mask = random_masks(dsa, B, T, 4)
    ln, dl = torch.tensor(lens, dtype=torch.int32, device=DEV), torch.tensor(drafts, dtype=torch.int32, device=DEV)
    o, lse = dsa.mla_sparse.forward_mqa_tree(q, cache, bt, ln, mask, SCALE, draft_lens=dl)
    assert o.dtype == served and o.shape == (B, T, H, 512) and lse.dtype == F32
    check_tree(o, lse, tree64(q.to(served), cache, bt, lens, mask, drafts, SCALE), fmt)
    for k in range(4):
        o2, lse2 = dsa.mla_sparse.forward_mqa_tree(q.to(served).view(B * T, H, 576) if k == 3 else q, cache,
                                                   bt.long() if k != 1 else bt, ln.long() if k != 2 else ln, mask, SCALE,
                                                   draft_lens=dl.long() if k else dl)
        assert torch.equal(o2.view_as(o), o) and torch.equal(lse2.view_as(lse), lse)
    with pytest.raises(RuntimeError):
        dsa.mla_sparse.forward_mqa_tree(q, cache, bt, ln.float(), mask, SCALE)


@pytest.mark.parametrize("lens,amp,step", [([32768, 32000], 1.0, 2.0 ** -16), ([32769, 33000], 1.0, 2.0 ** -11),
                                           ([1500, 9001], 0.25, 5 * 2.0 ** -17), ([1024, 700], 0.25, 2.0 ** -22)])
def test_tree_lse_of_peaked_rows(dsa, oracle, lens, amp, step):
    """Queries so large that a key or two carry each row, so that lse keeps the error
    of their scores. An fp8 key's value is held to `step` of itself: two products to a
    score up to 32768 positions, one beyond, scales of 2^-10 to 2^-8 (amp 1/4: N(0, 1)
    rows have 2^-7.9 to 2^-6.6) cut less finely, up to 1024 positions the first
    product's own remainder. In the 2-norm that leaves step / sqrt 3 of the latent
    part's terms. The f32 accumulator cuts each of the up to 1152 products below a
    quarter of its last place, 2^-25 of a partial sum, and those are taken as no larger
    than twice the score; each of the 72 instructions rounds the sum once, 2^-23."""
    B, T, H = len(lens), 2, 16
    bt, pages = tables(lens, 64, 41)
    cache = make_cache("fp8", pages, 64, 42, oracle)
    rows = cache.view(-1, 656)
    rows[:, 512:528] = (rows[:, 512:528].contiguous().view(F32) * amp).view(torch.uint8)
    q = (torch.randn(B, T, H, 576, generator=gen(43), device=DEV) * 16.0).to(BF)
    mask = random_masks(dsa, B, T, 44)
    o, lse = torch.empty(B, T, H, 512, dtype=BF, device=DEV), torch.empty(B, T, H, device=DEV)
    dsa.tree_mla_decode(o, lse, q, cache, bt, torch.tensor(lens, dtype=torch.int32, device=DEV), mask, SCALE)
    ref = tree64(q, cache, bt, lens, mask, None, SCALE)
    check_tree(o, lse, ref, "fp8")
    k2 = values64(cache)[:, :512].square().mean(0)
    norm = (q[..., :512].double().square() @ k2).sqrt().max() * SCALE
    rms = (lse.double() - ref[1]).square().mean().sqrt()
    tol = float(step / 3 ** 0.5 * norm) + float(ref[1].abs().max()) * 2 * (1152 * 2.0 ** -25 + 72 * 2.0 ** -23)
    assert float(rms) <= tol, (float(rms), tol)


@pytest.mark.parametrize("wide", [576, 580, 2000])
def test_gather_into_one_row_of_any_stride(dsa, oracle, wide):
    """A single output row's stride says nothing of its alignment."""
    cache = make_cache("fp8", 2, 64, 2, oracle)
    bt = torch.tensor([[1]], dtype=torch.int32, device=DEV)
    buf = torch.full((1, wide), 9.0, dtype=BF, device=DEV)
    dsa.gather_cache(buf[:, :576], cache, bt, torch.tensor([0, 1], dtype=torch.int32, device=DEV))
    assert torch.equal(buf[:, :576], plain_rows(cache, BF)[64:65]) and bool((buf[:, 576:] == 9).all())
