"""Log probabilities of given tokens, entropies and alternatives against plain formulas in 64 bits.

Tolerances.  A result is built from m (a logit, exact), s and u.  The terms exp(x - m) are off by a few units of 2^-24 times
(1 + |x - m|), for |x - m| up to 20 (what is further down adds less than 2e-9) at most 4e-6 each with any sign, and a sum of V terms kept in V / 512 steps
and joined over threads by up to V / 512 * 2^-24 relative (2e-5 at 160,000 would be the bound if all had one sign; rounding to nearest leaves its
root, 1e-6).  So ln s and u / s are off by about 5e-6 times 1 + their size, and 2e-5 * (1 + |result|) holds every case with a margin;
ids have no tolerance at all."""
import math

import numpy as np
import pytest
import torch

DEV = "cuda"


def plain(x, tokens, k):
    """x: float64 [n, V] on the CPU."""
    n, V = x.shape
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    m = x.amax(1, keepdim=True)
    some = (m > -math.inf)[:, 0]
    d = torch.where(x > -math.inf, x - torch.where(m > -math.inf, m, torch.zeros_like(m)), torch.full_like(x, -math.inf))
    e = torch.exp(d)
    s = e.sum(1)
    ln_s = torch.log(s)
    lse = torch.where(some, m[:, 0] + ln_s, torch.full_like(ln_s, -math.inf))
    H = torch.where(some, ln_s - torch.where(e > 0, e * d, torch.zeros_like(e)).sum(1) / s, torch.zeros_like(s))
    lp = torch.where(some[:, None], d - torch.where(some, ln_s, torch.zeros_like(s))[:, None], torch.full_like(x, -math.inf))
    t = tokens.long()
    got = torch.where((t >= 0) & (t < V), lp.gather(1, t.clamp(0, V - 1)[:, None])[:, 0], torch.full((n,), -math.inf, dtype=torch.float64))
    order = torch.from_numpy(np.argsort(-x.numpy(), axis=1, kind="stable")[:, :k].copy())      # equal logits by ascending id
    return got, H, lse, order, lp.gather(1, order)


def call(logits, tokens, k, rows=None, err=None):
    from airun_b200.kernels import ops
    n = tokens.shape[0]
    lp, H, lse = (torch.full((n,), 7.0, device=DEV) for _ in range(3))
    ids = torch.full((n, k), -7, dtype=torch.int32, device=DEV) if k else None
    tops = torch.full((n, k), 7.0, device=DEV) if k else None
    ops.token_logprobs(logits, tokens, lp, H, lse, ids, tops, rows=rows, err=err)
    torch.cuda.synchronize()
    return [None if t is None else t.cpu() for t in (lp, H, lse, ids, tops)]


def near(got, want, tol=2e-5):
    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)) and torch.equal(got[~fine], want[~fine]), (got[~fine], want[~fine])
    off = (got[fine] - want[fine]).abs() / (1 + want[fine].abs())
    assert off.numel() == 0 or float(off.max()) <= tol, float(off.max())


def check(logits, tokens, k, rows=None, tol=2e-5):
    got = call(logits, tokens, k, rows)
    x = (logits if rows is None else logits[rows.long()]).double().cpu()[: tokens.shape[0]]
    want = plain(x, tokens.cpu(), k)
    for g, w in zip(got[:3], want[:3]):
        near(g, w, tol)
    if k:
        assert torch.equal(got[3].long(), want[3])
        near(got[4], want[4], tol)
    return got


def some_tokens(n, V, seed):
    t = torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    if n > 2:
        t[1], t[2] = -1, V                            # a padded row, an id behind the vocabulary
    return t.to(DEV)


SIZES = [(1, 1, 1), (3, 2, 2), (5, 31, 31), (4, 129, 128), (7, 384, 5), (2, 2047, 9), (2, 2048, 40), (2, 2049, 8), (3, 4099, 3), (1, 8192, 1), (1, 16411, 20),
         (9, 50001, 33), (1, 151936, 5), (40, 65537, 128), (300, 5000, 20), (700, 1000, 0), (149, 33000, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,V,k", SIZES)
def test_tokens_against_64_bits(n, V, k, dtype):
    g = torch.Generator().manual_seed(n * 7919 + V)
    x = (torch.randn(n, V, generator=g) * 3).to(dtype).to(DEV)     # bfloat16: many equal logits
    check(x, some_tokens(n, V, V), k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pad,lead", [(1, 0), (3, 1), (5, 3), (8, 7)])
def test_tokens_any_stride_and_alignment(dtype, pad, lead):
    g = torch.Generator().manual_seed(pad)
    buf = torch.full((6, 9000 + pad + lead), 99.0)                 # what lies between the rows must not be read as a logit
    buf[:, lead:lead + 9000] = torch.randn(6, 9000, generator=g)
    x = buf.to(dtype).to(DEV)[:, lead:lead + 9000]
    check(x, some_tokens(6, 9000, pad), 11)
    check(x[:1], some_tokens(1, 9000, pad), 11)
    check(x[:, :700], some_tokens(6, 700, pad), 11)


@pytest.mark.gpu
def test_tokens_of_picked_rows_and_bad_rows():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(12, 6000, generator=g).to(DEV)
    rows = torch.tensor([11, 0, 7, 7, 3], dtype=torch.int32, device=DEV)                 # one row twice, for two tokens
    check(x, some_tokens(5, 6000, 4), 4, rows=rows)
    from airun_b200.kernels import ops
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    rows = torch.tensor([2, -1, 12], dtype=torch.int32, device=DEV)
    lp, H, lse, ids, tops = call(x, some_tokens(3, 6000, 4).clamp(0, 5999), 4, rows, err)
    assert math.isfinite(lp[0]) and lp[1:].tolist() == [-math.inf] * 2 and H[1:].tolist() == [0.0, 0.0] and lse[1:].tolist() == [-math.inf] * 2
    assert ids[1:].tolist() == [[-1] * 4] * 2 and tops[1:].tolist() == [[-math.inf] * 4] * 2
    assert int(err.item()) == 16 and "row" in ops.describe_device_error(16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [300, 7001, 70001])
def test_tokens_masks_ties_and_not_a_number(dtype, V):
    low = torch.finfo(dtype).min
    g = torch.Generator().manual_seed(V)
    x = torch.randn(14, V, generator=g)
    x[0] = -math.inf                                   # nothing is left
    x[1] = math.nan
    x[2] = 0.0                                         # all equal
    x[3] = low                                         # all at the type's lowest value: still a distribution
    x[4, 5:] = -math.inf                               # fewer than k
    x[5, : V - 3] = low
    x[6, ::2] = math.nan
    x[7, 17] = math.inf
    x[8] = -0.0
    x[8, ::3] = 0.0                                    # zeros of both signs are equal
    x[9] = torch.arange(V) * (60.0 / V)                # sorted
    x[10] = -torch.arange(V) * (60.0 / V)
    x[11] *= 1000.0                                    # far apart
    x[12, V // 2:] = torch.finfo(dtype).max
    x[13] = (torch.arange(V) % 512 == 3).float() * 5   # the largest ones repeat at the threads' stride
    x = x.to(dtype).to(DEV)
    t = torch.full((14,), 4, dtype=torch.int32, device=DEV)
    keep = [i for i in range(14) if i != 7]
    for k in (0, 1, 7, 32, 100):
        check(x[keep].contiguous(), t[keep], k)
        lp, H, lse, ids, tops = call(x[7:8].contiguous(), t[7:8], k)
        assert lp[0] == -math.inf and math.isnan(H[0]) and lse[0] == math.inf
        if k:
            assert ids[0, 0] == 17 and math.isnan(tops[0, 0]) and bool((tops[0, 1:] == -math.inf).all())
    one = torch.full((1, V), -math.inf)
    one[0, V - 2] = 3.0
    got = check(one.to(dtype).to(DEV), torch.tensor([V - 2], dtype=torch.int32, device=DEV), 3)
    assert got[0][0] == 0.0 and got[1][0] == 0.0 and got[3][0].tolist() == [V - 2, 0, 1]


@pytest.mark.gpu
def test_tokens_rows_far_into_a_large_buffer():
    """Row 17,000 of 131,072 columns lies behind 2^31 elements."""
    V = 131072
    x = torch.empty(17001, V, dtype=torch.bfloat16, device=DEV)
    x[17000] = torch.randn(V, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    rows = torch.tensor([17000], dtype=torch.int32, device=DEV)
    got = call(x, torch.tensor([77], dtype=torch.int32, device=DEV), 6, rows)
    want = plain(x[17000:].double().cpu(), torch.tensor([77]), 6)
    near(got[0], want[0])
    assert torch.equal(got[3].long(), want[3])


@pytest.mark.gpu
def test_tokens_leave_rows_behind_the_last_alone_and_repeat_bit_for_bit():
    from airun_b200.kernels import ops
    x = torch.randn(30, 20000, generator=torch.Generator().manual_seed(5)).to(DEV)
    t = some_tokens(30, 20000, 1)
    lp, ids, tops = torch.full((40,), 7.0, device=DEV), torch.full((40, 3), -7, dtype=torch.int32, device=DEV), torch.full((40, 3), 7.0, device=DEV)
    kept = []
    for _ in range(3):
        ops.token_logprobs(x, t, lp[:30], top_ids=ids[:30], top_logprobs=tops[:30])
        kept.append((lp.clone(), ids.clone(), tops.clone()))
    assert lp[30:].unique().tolist() == [7.0] and ids[30:].unique().tolist() == [-7] and tops[30:].unique().tolist() == [7.0]
    for got in kept[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got, kept[0]))
    ops.token_logprobs(x[:0], t[:0], lp[:0])            # no rows: nothing happens


@pytest.mark.gpu
def test_tokens_on_another_stream_and_in_two_graphs():
    from airun_b200.kernels import ops
    x = torch.randn(6, 40000, generator=torch.Generator().manual_seed(8)).to(DEV)
    t = some_tokens(6, 40000, 2)
    want = call(x, t, 5)
    places = [(torch.empty(6, device=DEV), torch.empty(6, 5, dtype=torch.int32, device=DEV), torch.empty(6, 5, device=DEV)) for _ in range(2)]
    graphs = []
    torch.cuda.synchronize()
    for lp, ids, tops in places:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.token_logprobs(x, t, lp, top_ids=ids, top_logprobs=tops)
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for lp, ids, tops in places:
        assert torch.equal(lp.cpu(), want[0]) and torch.equal(ids.cpu(), want[3]) and torch.equal(tops.cpu(), want[4])


# ---------------------------------------------------------------- from hidden states
def head(h, w, tokens, k, scale=1.0, cap=None, ws=None, **kw):
    from airun_b200.kernels import ops
    n = h.shape[0]
    lp, H, lse = (torch.full((n,), 7.0, device=DEV) for _ in range(3))
    ids = torch.full((n, k), -7, dtype=torch.int32, device=DEV) if k else None
    tops = torch.full((n, k), 7.0, device=DEV) if k else None
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.head_logprobs(h, w, tokens, lp, err, H, lse, ids, tops, scale=scale, soft_cap=cap, ws=ws)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    return [None if t is None else t.cpu() for t in (lp, H, lse, ids, tops)]


def grid_inputs(n, H, V, dtype, seed):
    """Multiples of 1/4 up to 1 and of 1/64 up to 1/8: every sum of up to 8,192 products is a multiple of 1/256 below 1,024 and
    exact in 32 bits in any order, so the logits have no rounding and many of them are equal."""
    g = torch.Generator().manual_seed(seed)
    h = torch.randint(-4, 5, (n, H), generator=g).float() / 4
    w = torch.randint(-8, 9, (V, H), generator=g).float() / 64
    return h.to(dtype).to(DEV), w.to(dtype).to(DEV)


HEAD_SIZES = [(1, 64, 1, 1), (1, 8, 300, 3), (2, 4096, 5000, 5), (5, 72, 257, 16), (8, 1024, 20000, 0), (64, 200, 4000, 4), (100, 512, 16400, 1), (127, 64, 384, 3),
              (128, 1032, 33, 16), (129, 520, 1000, 2), (256, 96, 2049, 5), (257, 2048, 1500, 8), (700, 1024, 20000, 0), (1111, 64, 700, 2), (3, 64, 160000, 7),
              (300, 136, 40000, 16), (5, 256, 5000, 40), (200, 72, 3001, 100)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,H,V,k", HEAD_SIZES)
def test_head_exact_logits(n, H, V, k, dtype):
    h, w = grid_inputs(n, H, V, dtype, n + H + V)
    t = some_tokens(n, V, n)
    got = head(h, w, t, k)
    want = plain(h.double().cpu() @ w.double().cpu().t(), t.cpu(), k)
    for g, x in zip(got[:3], want[:3]):
        near(g, x)
    if k:
        assert torch.equal(got[3].long(), want[3])
        near(got[4], want[4])


def off_by(h, w, steps):
    """How far a logit may be off: ``steps`` additions, each cut off at a unit (2^-23) of a sum that no partial sum exceeds."""
    return steps * 2.0 ** -23 * float((h.abs() @ w.abs().t()).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,H,V,scale,cap", [(3, 4096, 9000, 1.0, None), (130, 2048, 6000, 0.5, None), (64, 1024, 5001, 1.0, 30.0), (260, 776, 3000, 2.0, 5.0),
                                             (20, 100, 900, -1.5, 8.0), (70, 33, 500, 1.0, None)])
def test_head_rounded_logits(n, H, V, scale, cap, dtype):
    """Sums in parts of 512 values: 32 steps of 16 and the parts; float32 sums, and bfloat16 ones of widths that no tensor map takes, value by value.
    The logits' errors reach a log probability at most twice (its own, the sum's), an entropy at most 2 ln V times; a cap shrinks them, tanh
    itself is off by 2^-22 of the cap."""
    g = torch.Generator().manual_seed(n)
    h, w = torch.randn(n, H, generator=g).to(dtype).to(DEV), (0.05 * torch.randn(V, H, generator=g)).to(dtype).to(DEV)
    t = some_tokens(n, V, n)
    x = h.double().cpu() @ w.double().cpu().t() * scale
    off = abs(scale) * off_by(h.double().cpu(), w.double().cpu(), H if dtype == torch.float32 or H % 8 else min(H, 512) / 16 + H / 512)
    if cap is not None:
        x, off = cap * torch.tanh(x / cap), off + cap * 2.0 ** -22
    want = plain(x, t.cpu(), 4)
    got = head(h, w, t, 4, scale, cap)
    tol = 2e-5 + off * (2 + 2 * math.log(V))
    for a, b in zip(got[:3], want[:3]):
        near(a, b, tol)
    near(got[4], want[4], tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_head_strided_operands_and_neighbours_left_alone(dtype):
    from airun_b200.kernels import ops
    h, w = grid_inputs(150, 128, 3000, dtype, 4)
    hb, wb = torch.full((150, 144), 50.0, dtype=dtype, device=DEV), torch.full((3000, 136), 50.0, dtype=dtype, device=DEV)
    hb[:, 8:136], wb[:, :128] = h, w
    t = some_tokens(150, 3000, 5)
    want = plain(h.double().cpu() @ w.double().cpu().t(), t.cpu(), 5)
    lp, ids, tops = torch.full((160,), 7.0, device=DEV), torch.full((160, 5), -7, dtype=torch.int32, device=DEV), torch.full((160, 5), 7.0, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.head_logprobs(hb[:, 8:136], wb[:, :128], t, lp[:150], err, top_ids=ids[:150], top_logprobs=tops[:150])
    near(lp[:150].cpu(), want[0])
    assert torch.equal(ids[:150].cpu().long(), want[3]) and int(err.item()) == 0
    assert lp[150:].unique().tolist() == [7.0] and ids[150:].unique().tolist() == [-7] and tops[150:].unique().tolist() == [7.0]
    ops.head_logprobs(h[:0], w, t[:0], lp[:0], err)     # no rows: nothing happens


@pytest.mark.gpu
@pytest.mark.parametrize("n", [4, 140])
def test_head_rows_that_are_not_finite(n):
    """A hidden row of NaN, and weights that give -inf or NaN logits for some tokens."""
    h, w = grid_inputs(n, 64, 900, torch.bfloat16, 9)
    h[:, 0] = 1.0
    h[1] = math.nan
    w[100:900, 0] = -math.inf
    w[7, 3] = math.nan
    x = h.double().cpu() @ w.double().cpu().t()
    t = torch.full((n,), 5, dtype=torch.int32, device=DEV)
    for k in (3, 16, 100):
        want, got = plain(x, t.cpu(), k), head(h, w, t, k)
        for a, b in zip(got[:3], want[:3]):
            near(a, b)
        assert torch.equal(got[3].long(), want[3])
    w[100:900, 0] = math.inf
    w[7, 3] = 0.0
    got = head(h, w, t, 3)
    assert got[0][0] == -math.inf and math.isnan(got[1][0]) and got[2][0] == math.inf and got[3][0, 0] == 100


@pytest.mark.gpu
@pytest.mark.parametrize("n,V,k", [(4, 6000, 5), (300, 6000, 2), (3, 500, 40)])
def test_head_on_another_stream_and_in_two_graphs(n, V, k):
    from airun_b200.engine.batch import Workspace
    from airun_b200.kernels import ops
    h, w = grid_inputs(n, 256, V, torch.bfloat16, 2)
    t = some_tokens(n, V, 2)
    want = head(h, w, t, k)
    places, graphs = [], []
    for _ in range(2):
        places.append((torch.empty(n, device=DEV), torch.empty(n, k, dtype=torch.int32, device=DEV), torch.empty(n, k, device=DEV),
                       torch.zeros(1, dtype=torch.int32, device=DEV), Workspace(torch.device(DEV), 1 << 20)))
    for lp, ids, tops, err, ws in places:
        for captured in (False, True):
            ws.reset()
            if not captured:
                ops.head_logprobs(h, w, t, lp, err, top_ids=ids, top_logprobs=tops, ws=ws)
                torch.cuda.synchronize()
                lp.fill_(7.0)
                torch.cuda.synchronize()
                continue
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                ops.head_logprobs(h, w, t, lp, err, top_ids=ids, top_logprobs=tops, ws=ws)
            graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for lp, ids, tops, err, _ in places:
        assert torch.equal(lp.cpu(), want[0]) and torch.equal(ids.cpu(), want[3]) and torch.equal(tops.cpu(), want[4]) and int(err.item()) == 0


@pytest.mark.gpu
def test_head_sizes_that_fill_rounds_of_blocks_unevenly():
    """Rows and ids just off the tiles' and ranges' borders, on single SMs and on pairs."""
    for n, H, V, k in ((129, 64, 2368, 2), (255, 128, 16 * 148 + 1, 3), (385, 1024, 256 * 37 + 1, 2), (513, 64, 255, 4), (1024, 1088, 256 * 18, 0), (1025, 1024, 5000, 16)):
        h, w = grid_inputs(n, H, V, torch.bfloat16, n)
        t = some_tokens(n, V, n)
        got, want = head(h, w, t, k), plain(h.double().cpu() @ w.double().cpu().t(), t.cpu(), k)
        for g, x in zip(got[:3], want[:3]):
            near(g, x)
        assert k == 0 or torch.equal(got[3].long(), want[3]), (n, H, V)


@pytest.mark.gpu
@pytest.mark.parametrize("n,V,k", [(40, 70000, 16), (128, 70000, 8), (40, 70000, 0)])
def test_head_tiles_that_end_inside_a_warps_ids(n, V, k):
    """Tiles of 240 ids, whose last 16 share 32 columns with what lies behind: tokens at the start of the next tile belong to other warps, which come there early
    where every id of the one enters its lists and none of the other's does."""
    from airun_b200.kernels.fast import plan_head
    pair, ranges, tiles, bn, _ = plan_head(n, V, 64)
    assert not pair and tiles > 1 and bn % 64 == 48
    place = torch.arange(V) % (tiles * bn)
    late = place % bn // 32 % 2 == 1
    g = torch.Generator().manual_seed(7)
    h, w = torch.zeros(n, 64, dtype=torch.bfloat16), torch.randint(-8, 9, (V, 64), generator=g).to(torch.bfloat16) / 64
    h[:, 0], h[:, 1] = 1.0, torch.arange(n) % 5 / 4
    w[:, 0] = torch.where(late, (place // 2).float() / 16, torch.tensor(-4.0)).to(torch.bfloat16)
    first = torch.randint(0, ranges - 1, (n,), generator=g) * tiles * bn + bn
    t = (first + torch.randint(0, 16, (n,), generator=g)).to(torch.int32).to(DEV)
    want, got = plain(h.double() @ w.double().t(), t.cpu(), k), head(h.to(DEV), w.to(DEV), t, k)
    for a, b in zip(got[:3], want[:3]):
        near(a, b)
    if k:
        assert torch.equal(got[3].long(), want[3])


@pytest.mark.gpu
@pytest.mark.parametrize("n,H,V,k", [(1, 8, 1, 1), (1, 64, 129, 128), (9, 520, 1184, 20), (15, 136, 18944, 0), (16, 1032, 18945, 128), (17, 256, 7, 7), (24, 264, 37889, 5),
                                     (25, 72, 2049, 17), (31, 4104, 1300, 3), (32, 512, 50001, 16)])
def test_head_few_rows(n, H, V, k):
    """Ranges and tiles of every kind: one id, odd ones, last tiles and K-steps that are partly or wholly outside; the same bits again."""
    h, w = grid_inputs(n, H, V, torch.bfloat16, n * H + V)
    h[n // 2] = 0
    t = some_tokens(n, V, n)
    got, again = head(h, w, t, k, 0.5, 2.0), head(h, w, t, k, 0.5, 2.0)
    x = 2.0 * torch.tanh(0.5 * (h.double().cpu() @ w.double().cpu().t()) / 2.0)
    want = plain(x, t.cpu(), k)
    for a, b in zip(got[:3], want[:3]):
        near(a, b)
    if k:
        near(got[4], want[4])
        plainly = head(h, w, t, k)
        exact = plain(h.double().cpu() @ w.double().cpu().t(), t.cpu(), k)
        assert torch.equal(plainly[3].long(), exact[3])
        near(plainly[4], exact[4])
    for a, b in zip(got, again):
        assert a is None or torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3, 20])
def test_head_few_rows_infinite_logits_stay_so(n):
    """An infinite product early in a sum, with parts behind it; of both signs: no number."""
    h, w = grid_inputs(n, 1024, 700, torch.bfloat16, 21)
    h[:, 3], h[:, 900] = 1.0, 1.0
    w[5, 3], w[6, 3], w[7, 900] = math.inf, -math.inf, -math.inf
    w[8, 3], w[8, 900] = -math.inf, math.inf
    t = torch.tensor([5, 6, 8] + [9] * (n - 3), dtype=torch.int32, device=DEV)
    got = head(h, w, t, 2)
    assert bool((got[2] == math.inf).all()) and bool(torch.isnan(got[1]).all()) and bool((got[3][:, 0] == 5).all())
    w[5, 3] = 0.0
    want, got = plain(h.double().cpu() @ w.double().cpu().t(), t.cpu(), 3), head(h, w, t, 3)
    for a, b in zip(got[:3], want[:3]):
        near(a, b)
    assert got[0][1] == -math.inf and got[0][2] == -math.inf and torch.equal(got[3].long(), want[3])


@pytest.mark.gpu
def test_head_few_and_more_rows_agree():
    """The last rows of the one form and the first of the other: the same rows, alone and among others."""
    h, w = grid_inputs(33, 1024, 9001, torch.bfloat16, 11)
    t = some_tokens(33, 9001, 3)
    few, more = head(h[:32], w, t[:32], 5), head(h, w, t, 5)
    for a, b in zip(few[:3], more[:3]):
        near(a, b[:32].double())
    assert torch.equal(few[3], more[3][:32])


@pytest.mark.gpu
def test_head_few_rows_far_into_a_large_vocabulary():
    """Rows of a strided weight past 2^31 elements; the last ids lead."""
    V, H = 300000, 64
    buf = torch.zeros(V, 8192, dtype=torch.bfloat16, device=DEV)
    w = buf[:, 8000:8000 + H]
    g = torch.Generator().manual_seed(5)
    w.copy_((torch.randint(-8, 9, (V, H), generator=g).float() / 64).to(torch.bfloat16))
    h, _ = grid_inputs(6, H, 8, torch.bfloat16, 6)
    t = torch.tensor([0, V - 1, V - 2, V, -1, 149999], dtype=torch.int32, device=DEV)
    want, got = plain(h.double().cpu() @ w.double().cpu().t(), t.cpu(), 4), head(h, w, t, 4)
    for a, b in zip(got[:3], want[:3]):
        near(a, b)
    assert torch.equal(got[3].long(), want[3])


def test_plan_of_few_rows_covers_the_vocabulary():
    from airun_b200.kernels.fast import plan_few
    for V in list(range(1, 2500)) + [18944, 18945, 32000, 151936, 262144, 1 << 20]:
        for sms in (148, 132, 2):
            tiles, bn = plan_few(V, sms)
            assert 8 <= bn <= 128 and tiles >= 1 and -(-V // (tiles * bn)) <= sms, (V, sms)


@pytest.mark.gpu
def test_head_calls_on_two_streams_with_workspaces_of_their_own():
    from airun_b200.engine.batch import Workspace
    from airun_b200.kernels import ops
    sets = []
    for i, (n, V) in enumerate(((70, 9000), (3, 20000))):
        h, w = grid_inputs(n, 256, V, torch.bfloat16, i)
        t = some_tokens(n, V, i)
        sets.append((h, w, t, torch.empty(n, device=DEV), torch.empty(n, 6, dtype=torch.int32, device=DEV), torch.empty(n, 6, device=DEV),
                     torch.zeros(1, dtype=torch.int32, device=DEV), Workspace(torch.device(DEV), 1 << 20), torch.cuda.Stream(),
                     plain(h.double().cpu() @ w.double().cpu().t(), t.cpu(), 6)))
    torch.cuda.synchronize()
    for _ in range(20):
        for h, w, t, lp, ids, tops, err, ws, stream, _ in sets:
            with torch.cuda.stream(stream):
                ws.reset()
                ops.head_logprobs(h, w, t, lp, err, top_ids=ids, top_logprobs=tops, ws=ws)
    torch.cuda.synchronize()
    for h, w, t, lp, ids, tops, err, ws, stream, want in sets:
        near(lp.cpu(), want[0])
        assert torch.equal(ids.cpu().long(), want[3]) and int(err.item()) == 0


def test_plan_of_ranges_covers_the_vocabulary():
    """Every id lies in one range, no range is empty, tiles have a width the products take."""
    import random
    from airun_b200.kernels.fast import plan_head
    rng = random.Random(1)
    for _ in range(3000):
        n, V, K = int(2 ** rng.uniform(0, 18)), int(2 ** rng.uniform(0, 18)), 8 * int(2 ** rng.uniform(0, 10))
        pair, ranges, tiles, bn, part = plan_head(n, V, K, rng.choice((148, 132, 20, 2)))
        assert ranges * tiles * bn >= V > (ranges - 1) * tiles * bn and 16 <= bn <= 256 and bn % (32 if pair else 16) == 0 and part in (2, 8), (n, V, K)
        assert not pair or n > 128


class _Fake:
    """A tensor's stand-in that says it is on the GPU, for the checks that come before any launch."""

    def __new__(cls, *shape, dtype=torch.float32):
        t = torch.empty(*shape, dtype=dtype)

        class OnGpu(torch.Tensor):
            is_cuda = True
        return t.as_subclass(OnGpu)


def test_refusals(monkeypatch):
    from airun_b200.kernels import ops
    monkeypatch.setattr(ops, "_fn", lambda *a, **k: pytest.fail("launched"))
    monkeypatch.setattr(ops, "_here", ops._cuda)
    x, t, lp = _Fake(4, 100), _Fake(4, dtype=torch.int32), _Fake(4)

    def refused(match, logits=x, tokens=t, logprob=lp, **kw):
        with pytest.raises(ops.KernelError, match=match):
            ops.token_logprobs(logits, tokens, logprob, **kw)

    refused("GPU", logits=torch.empty(4, 100))
    refused("int32", tokens=_Fake(4, dtype=torch.int64))
    refused("float32", logprob=_Fake(3))
    refused("float32", entropy=_Fake(4, dtype=torch.float64))
    refused("every token", logits=_Fake(3, 100))
    refused("row-major", logits=_Fake(100, 4).t())
    refused("overlap", logits=_Fake(400).as_strided((4, 100), (50, 1)))
    refused("together", top_ids=_Fake(4, 3, dtype=torch.int32))
    refused("to the vocabulary", top_ids=_Fake(4, 101, dtype=torch.int32), top_logprobs=_Fake(4, 101))
    refused("to the vocabulary", logits=_Fake(4, 999), top_ids=_Fake(4, 129, dtype=torch.int32), top_logprobs=_Fake(4, 129))
    refused("one shape", top_ids=_Fake(4, 3, dtype=torch.int32), top_logprobs=_Fake(4, 2))
    refused("int32", rows=_Fake(5, dtype=torch.int32))
    refused("one row", rows=t, logits=_Fake(0, 100))
    monkeypatch.setattr(ops, "_fn", lambda *a, **k: (lambda *b: 0))
    refused("dtype", logits=_Fake(4, 100, dtype=torch.float16))


def test_head_refusals(monkeypatch):
    from airun_b200.kernels import ops
    monkeypatch.setattr(ops, "_fn", lambda *a, **k: pytest.fail("launched"))
    monkeypatch.setattr(ops, "_here", ops._cuda)
    h, w, t, lp, err = _Fake(4, 64), _Fake(100, 64), _Fake(4, dtype=torch.int32), _Fake(4), _Fake(1, dtype=torch.int32)

    def refused(match, hidden=h, weight=w, tokens=t, logprob=lp, err=err, **kw):
        with pytest.raises(ops.KernelError, match=match):
            ops.head_logprobs(hidden, weight, tokens, logprob, err, **kw)

    refused("GPU", hidden=torch.empty(4, 64))
    refused("do not agree", weight=_Fake(100, 72))
    refused("share a type", weight=_Fake(100, 64, dtype=torch.bfloat16))
    refused("row-major", hidden=_Fake(64, 4).t())
    refused("token for every row", tokens=_Fake(3, dtype=torch.int32))
    refused("int32", tokens=_Fake(4, dtype=torch.int64))
    refused("float32", logprob=_Fake(4, 1))
    refused("together", top_logprobs=_Fake(4, 3))
    refused("to the vocabulary", top_ids=_Fake(4, 101, dtype=torch.int32), top_logprobs=_Fake(4, 101))
    refused("int32", err=_Fake(1))
    refused("overlap", hidden=_Fake(64).as_strided((4, 64), (0, 1)))
    refused("overlap", weight=_Fake(6400).as_strided((100, 64), (32, 1)))
    for scale in (float("nan"), float("inf"), 1e39):
        refused("finite", scale=scale)
    for cap in (0.0, -1.0, 1e-50, 1e39, float("nan")):
        refused("positive", soft_cap=cap)
    refused("dtype", hidden=_Fake(4, 64, dtype=torch.float16), weight=_Fake(100, 64, dtype=torch.float16))


# ---------------------------------------------------------------- nearly all of a row's probability on one token
APART = (14.0, 16.125, 18.25)          # exact in bfloat16: the second token has 8e-7, 1e-7 and 1.2e-8
# The leading logit is 0, so differences are exact.  exp(-d): d * log2(e) is rounded twice, each time by 2^-24 of up to 18.25 in natural units, and the
# exponential is off by 2^-22 of itself: 2.4e-6 in all; a handful of roundings of the sums, log1p and the quotient are 4e-7.
PEAKED = 3e-6


def near_relatively(got, want, also=0.0):
    assert bool(((got.double() - want).abs() <= PEAKED * want.abs() + also).all()), (got, want)


def check_peaked(got, apart, leads, also=0.0):
    """Rows whose only logits are 0 and -apart; ``leads``: which rows ask for the leading token; ``also``: an absolute error that is allowed besides."""
    d = torch.tensor(apart, dtype=torch.float64)
    e = torch.exp(-d)
    rest = torch.log1p(e)
    near_relatively(got[0], torch.where(leads, -rest, -d - rest), also)
    near_relatively(got[1], rest + d * e / (1 + e), also)
    near_relatively(got[2], rest, also)
    near_relatively(got[4], torch.stack((-rest, -d - rest), 1), also if isinstance(also, float) else also[:, None])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,repeats", [(300, 1), (20000, 1), (20000, 3), (151936, 1)])
def test_tokens_peaked_rows_in_any_order(V, repeats, dtype):
    """The leading token before and behind the second one: in one batch of a thread, in a later one, in another thread or block."""
    places = [p for p in (1, 2, 70, 2049, 8193, V - 1) if p < V]
    rows = [(a, b, d) for a in places for b in places if a != b for d in APART] * repeats
    x = torch.full((len(rows), V), -math.inf)
    for r, (a, b, d) in enumerate(rows):
        x[r, a], x[r, b] = 0.0, -d
    leads = torch.arange(len(rows)) % 2 == 0
    t = torch.tensor([a if r % 2 == 0 else b for r, (a, b, d) in enumerate(rows)], dtype=torch.int32, device=DEV)
    got = call(x.to(dtype).to(DEV), t, 2)
    check_peaked(got, [d for _, _, d in rows], leads)
    assert got[3].tolist() == [[a, b] for a, b, _ in rows]
    for g, w in zip(call(x.to(dtype).to(DEV), t, 0)[:3], got[:3]):
        near_relatively(g, w.double())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [5, 40, 100, 300])
def test_head_peaked_rows_in_any_order(n):
    """The same from hidden states, every row one column of the weights: in the 32 ids a thread takes at a time, in later ones, in another tile or range.  Among the
    32 that hold the leading one the others are rounded to 2^-24 of its 1 (twice at most) where the logits are never written."""
    V = 20000
    pairs = [(1, 2), (2, 1), (1, 70), (70, 1), (1, 40), (40, 1), (1, 300), (300, 1), (3, 19990), (19990, 3), (64, 129), (129, 64)]
    w = torch.full((V, 64), -2000.0)
    apart = [APART[j % 3] for j in range(len(pairs))]
    for j, (a, b) in enumerate(pairs):
        w[a, j], w[b, j] = 0.0, -apart[j]
    at = [r % len(pairs) for r in range(n)]
    h = torch.zeros(n, 64)
    h[torch.arange(n), at] = 1.0
    leads = torch.arange(n) % 2 == 0
    t = torch.tensor([pairs[j][r % 2] for r, j in enumerate(at)], dtype=torch.int32, device=DEV)
    got = head(h.to(torch.bfloat16).to(DEV), w.to(torch.bfloat16).to(DEV), t, 2)
    together = torch.tensor([pairs[j][0] // 32 == pairs[j][1] // 32 and n > 32 for j in at])
    check_peaked(got, [apart[j] for j in at], leads, together * 2.0 ** -23)
    assert got[3].tolist() == [list(pairs[j]) for j in at]


# ---------------------------------------------------------------- the command that measures a model
def test_losses_of_places_are_worked_out_in_64_bits(monkeypatch):
    """To the last digits of 64 bits (a sum of 5,000 terms: 1e-13), in blocks of rows too; a logit that is not a number leaves its row without a loss."""
    from airun_b200 import cli
    g = torch.Generator().manual_seed(2)
    x = 5 * torch.randn(40, 5000, generator=g)
    x[3, 17] += 60.0                                   # one leading token: a loss of about 1e-20
    t = torch.randint(0, 5000, (40,), generator=g)
    t[3], t[4] = 17, int(x[4].argmax())
    losses, best = cli.place_losses(x, t.tolist())
    d = x.numpy().astype(np.longdouble) - x.numpy().max(1, keepdims=True).astype(np.longdouble)
    want = np.log(np.exp(d).sum(1)) - d[np.arange(40), t.numpy()]
    assert np.abs(np.array(losses) - want.astype(np.float64)).max() <= 1e-12
    assert best == [bool(x[i].argmax() == t[i]) for i in range(40)] and best[3] and best[4]
    x[5, 9] = math.nan
    x[6] = math.nan
    x[7, int(t[7])] = -math.inf
    losses, _ = cli.place_losses(x, t.tolist())
    assert math.isnan(losses[5]) and math.isnan(losses[6]) and losses[7] == math.inf and all(math.isfinite(v) for v in losses[:5] + losses[8:])
    monkeypatch.setattr(cli, "LOSS_BLOCK", 10001)      # two rows a block
    again, best_again = cli.place_losses(x, t.tolist())
    assert np.array_equal(again, losses, equal_nan=True) and best_again[:5] == best[:5]


def test_a_head_that_only_forms_logits_is_scored_in_blocks_of_rows(monkeypatch):
    """Head.score holds no more than HEAD_CHUNK logits, however many rows there are; every row meets its own token and place."""
    from types import SimpleNamespace
    from airun_b200.engine.batch import Workspace
    from airun_b200.kernels import ops
    from airun_b200.parts.base import Head, TokenScores
    g = torch.Generator().manual_seed(1)
    w = torch.randn(50, 8, generator=g)

    class Plain(Head):
        V = 50

        def forward(self, ctx, h, out):
            out.copy_(h @ w.t())

    def told(logits, tokens, logprob, entropy, lse, top_ids, top_logprobs):
        held.append(logits.numel())
        lp, H, _, ids, tops = plain(logits.double(), tokens, 3)
        for place, value in ((logprob, lp), (entropy, H), (top_ids, ids), (top_logprobs, tops)):
            if place is not None:
                place.copy_(value)

    monkeypatch.setattr(ops, "token_logprobs", told)
    for chunk, most in ((1 << 26, 23), (350, 7), (49, 1)):
        monkeypatch.setattr(ops, "HEAD_CHUNK", chunk)
        for top in (0, 3):
            held, h, t = [], torch.randn(23, 8, generator=g), torch.randint(0, 50, (23,), generator=g, dtype=torch.int32)
            ctx, scores = SimpleNamespace(ws_main=Workspace(torch.device("cpu"), 1 << 10)), TokenScores.empty(23, top, "cpu")
            Plain().score(ctx, h, t, scores)
            want = plain((h @ w.t()).double(), t, 3)
            near(scores.logprob, want[0]), near(scores.entropy, want[1])
            assert max(held) == most * 50 and sum(held) == 23 * 50 and ctx.ws_main.bytes() <= max(1 << 10, 4 * 50 * most + 256)
            if top:
                assert torch.equal(scores.top_ids.long(), want[3])
                near(scores.top_logprobs, want[4])


def test_a_bad_row_is_described_as_one_of_logits_too():
    from airun_b200.kernels import ops
    assert "row of logits" in ops.describe_device_error(16) and "expert" in ops.describe_device_error(16) and "segment" in ops.describe_device_error(16)


class _Huge:
    """The same as _Fake without memory: sizes that only the checks see."""

    def __new__(cls, *shape, dtype=torch.float32):
        class OnGpu(torch.Tensor):
            is_cuda = True
        return torch.empty(*shape, dtype=dtype, device="meta").as_subclass(OnGpu)


def test_refusals_of_sizes_beyond_32_bits_and_of_other_error_words(monkeypatch):
    """Numbers of rows, columns and tokens go to the kernels in 32 bits: what they would lose is refused, not cut off.  The device writes an int32 where the error word is."""
    from airun_b200.kernels import ops
    monkeypatch.setattr(ops, "_fn", lambda *a, **k: pytest.fail("launched"))
    monkeypatch.setattr(ops, "_here", ops._cuda)
    t, lp = _Fake(4, dtype=torch.int32), _Fake(4)
    for R, V in (((1 << 32) + 4, 10), (1 << 31, 1), (4, (1 << 32) + 10), (4, 1 << 31)):
        with pytest.raises(ops.KernelError, match="at most"):
            ops.token_logprobs(_Huge(R, V), t, lp)
    n = (1 << 32) + 2
    with pytest.raises(ops.KernelError, match="at most"):
        ops.token_logprobs(_Huge(4, 10), _Huge(n, dtype=torch.int32), _Huge(n), rows=_Huge(n, dtype=torch.int32))
    err = _Fake(1, dtype=torch.int32)
    for n, V, H in ((4, (1 << 32) + 16, 8), (4, 16, (1 << 32) + 8), ((1 << 32) + 1, 16, 8)):
        with pytest.raises(ops.KernelError, match="at most"):
            ops.head_logprobs(_Huge(n, H, dtype=torch.bfloat16), _Huge(V, H, dtype=torch.bfloat16), _Huge(n, dtype=torch.int32), _Huge(n), err)
    for bad in (_Fake(1), _Fake(1, dtype=torch.int64), _Fake(2, dtype=torch.int32), _Fake(0, dtype=torch.int32)):
        with pytest.raises(ops.KernelError, match="one int32"):
            ops.token_logprobs(_Fake(4, 100), t, lp, err=bad)


# ---------------------------------------------------------------- how exact the sums are
def peaked_hidden(n, H, V, seed):
    """Hidden rows whose logits have a spread of 1.3 and ten that stand out by 14 to 24 and less, as a trained model's do."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = (0.02 * torch.randn(V, H, generator=g, device=DEV))
    h = torch.randn(n, H, generator=g, device=DEV)
    ids = torch.randint(0, V, (n, 10), generator=g, device=DEV)
    lead = 14 + 10 * torch.rand(n, 1, generator=g, device=DEV) - (0.8 + 0.8 * torch.rand(n, 10, generator=g, device=DEV)).cumsum(1)
    rows = w[ids]
    h += torch.einsum("nl,nlh->nh", lead / rows.square().sum(-1), rows)
    return h.to(torch.bfloat16), w.to(torch.bfloat16), ids[:, 0].to(torch.int32)


def entropy_error(n, H, V, calls):
    """Root mean square over all rows of the entropies' relative errors against 64 bits."""
    off = []
    for seed in range(calls):
        h, w, t = peaked_hidden(n, H, V, 1000 * n + seed)
        got = head(h, w, t, 0)
        lp = torch.log_softmax(h.double() @ w.double().t(), dim=1)
        want = -(lp.exp() * lp).sum(1).cpu()
        off.append((got[1].double() - want) / want)
    return float(torch.cat(off).square().mean().sqrt())


@pytest.mark.gpu
@pytest.mark.parametrize("n,H,calls,limit", [(16, 4096, 4, 5.5e-7), (40, 4096, 4, 4e-6), (64, 4096, 4, 4e-6), (100, 4096, 4, 4e-6), (300, 4096, 2, 4e-6)])
def test_head_sums_stay_in_parts(n, H, calls, limit):
    """A logit near 20 is rounded to 2^-20 a step.  Up to 32 rows its parts of 64 and 128 values are added with compensation, so one such rounding is left, 3e-7 in the
    mean square (measured 3.4e-7; 8.7e-7 without compensation).  More rows add their parts of 128 and 512 values plainly: up to 32 roundings of partial sums on the way to 20,
    about 1e-6 (measured 0.9e-6 to 1.4e-6; one sum over all 4,096 values 1.1e-5).  An entropy of these rows is off by about what its leading logits are."""
    assert entropy_error(n, H, 12000, calls) <= limit


@pytest.mark.gpu
def test_head_whole_sums_would_be_seen(monkeypatch):
    """The measure above tells parts from one sum."""
    from airun_b200.kernels import fast
    plan = fast.plan_head
    monkeypatch.setattr(fast, "plan_head", lambda *a, **k: plan(*a, **k)[:4] + (64,))
    assert entropy_error(100, 4096, 12000, 2) > 4e-6


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 24, 200])
def test_tokens_beside_a_leading_one_are_summed_to_full_precision(n):
    """One token has all but about 1e-3 of a row, 151,935 others the rest.  Their terms' d = x - m is about -17: d * log2(e) is off by 1.3e-8 of itself (the constant
    as a float) and a rounding, which averages out, so terms by 2.3e-7; sums of terms of one sign, compensated and joined in a few steps, add about 1e-7.  Where a sum
    holds the leading token's 1 too each step rounds by up to 6e-8 of it, 6e-5 of what is looked for."""
    V, off = 151936, []
    for seed in range(-(-24 // n)):
        g = torch.Generator(device=DEV).manual_seed(7 * n + seed)
        x = 1.3 * torch.randn(n, V, generator=g, device=DEV)
        at = torch.randint(0, V, (n, 1), generator=g, device=DEV)
        x.scatter_(1, at, torch.logsumexp(x, 1, keepdim=True) + 6 + 2 * torch.rand(n, 1, generator=g, device=DEV))
        got = call(x, at[:, 0].to(torch.int32), 1)
        d = x.double() - x.double().amax(1, keepdim=True)
        rest = torch.where(d < 0, d.exp(), 0.0).sum(1)
        lp = -torch.log1p(rest)
        entropy = -lp - (d.exp() * d).sum(1) / (1 + rest)
        off.append(torch.stack(((got[0].double() - lp.cpu()) / lp.cpu(), (got[1].double() - entropy.cpu()) / entropy.cpu(), (got[4][:, 0].double() - lp.cpu()) / lp.cpu())))
    off = torch.cat(off, 1)
    assert float(off.square().mean(1).sqrt().max()) <= 4e-7 and float(off.abs().max()) <= 1e-6, (off.square().mean(1).sqrt(), off.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [16, 40, 100, 300])
def test_head_beside_a_leading_one(n):
    """The same from hidden states with exact logits: multiples of 1/8 from -14 to -18 under a leading 0, 20,000 ids.  A term: d * log2(e) is 20 to 26 and rounded by 2^-20
    at most, 6.6e-7 of the exponential, the constant is off by 1.3e-8 of itself, 2.4e-7 at 18, the exponential by 2^-22: 1.2e-6, the same for all ids of a logit, and
    2e-7 for the sums.  More than 32 rows also add the 31 ids beside the leading one to its 1, in two chains of 16 additions that each round by 2^-24 at most."""
    V, g = 20000, torch.Generator().manual_seed(n)
    w = torch.zeros(V, 64)
    w[:, :32] = -14 - torch.randint(0, 33, (V, 32), generator=g) / 8
    at = torch.randint(0, V, (32,), generator=g)
    w[at, torch.arange(32)] = 0.0
    col = torch.arange(n) % 32
    h = torch.zeros(n, 64)
    h[torch.arange(n), col] = 1.0
    got = head(h.to(torch.bfloat16).to(DEV), w.to(torch.bfloat16).to(DEV), at[col].to(torch.int32).to(DEV), 1)
    x = w.double().t()[col]
    rest = torch.where(x < 0, x.exp(), 0.0).sum(1)
    lp = -torch.log1p(rest)
    entropy = -lp - (x.exp() * x).sum(1) / (1 + rest)
    for found, want in ((got[0], lp), (got[1], entropy), (got[2], -lp), (got[4][:, 0], lp)):
        fine = ((found.double() - want).abs() <= 1.4e-6 * want.abs() + (2.0 ** -20 if n > 32 else 0.0)).all()
        assert bool(fine), float(((found.double() - want).abs() / want.abs()).max())


def test_plan_of_few_rows_leaves_room_for_three_stages():
    """A stage of head_few_kernel holds four K-steps of 64 values of a tile's ids and of the rows, in groups of eight; the products read 128 ids and 16 or 32 rows from
    the last ones on.  227 KB, of which one aligns the stages."""
    from airun_b200.kernels.fast import HEAD_FEW, plan_few
    up = lambda x: -(-x // 8) * 8      # noqa: E731
    for rows in range(1, HEAD_FEW + 1):
        for V in (1, 300, 2049, 20000, 32000, 50001, 128256, 151936, 262144):
            tiles, bn = plan_few(V, 148, rows)
            assert 1 <= bn <= 128 and -(-V // (tiles * bn)) <= 148
            beyond = 128 * ((16 if rows <= 16 else 32) - up(rows) + 128 - up(bn))
            assert 3 * 4 * 128 * (up(bn) + up(rows)) + beyond <= 230400 - 1024, (rows, V)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,n", [(301, 1), (2047, 3), (20003, 1), (20003, 5), (20003, 150), (70001, 1)])
def test_tokens_peaked_rows_that_start_and_end_between_vectors(V, n, dtype):
    """Leading and second tokens among the elements ahead of the first 16-byte boundary and behind the last one, which belong to the first and the last block; rows are
    picked, every one at another distance from a boundary, with large logits beside them."""
    places = [0, 1, 2, 6, 8, V - 9, V - 5, V - 2, V - 1]
    pairs = [(a, b, d) for a in places for b in places if a != b for d in APART[:1 + 2 * (n == 1)]]
    buf = torch.full((len(pairs), V + 5), 50.0)
    x = buf[:, 3:3 + V]
    x[:] = -math.inf
    for r, (a, b, d) in enumerate(pairs):
        x[r, a], x[r, b] = 0.0, -d
    x = buf.to(dtype).to(DEV)[:, 3:3 + V]
    g = torch.Generator().manual_seed(V)
    order = torch.randperm(len(pairs), generator=g).tolist()
    order = (order * (1 + n // len(order)))[:max(len(order) // n * n, n)]
    for at in range(0, len(order), n):
        rows = order[at:at + n]
        leads = torch.tensor([(at + i) % 2 == 0 for i in range(n)])
        t = torch.tensor([pairs[r][0 if leads[i] else 1] for i, r in enumerate(rows)], dtype=torch.int32, device=DEV)
        got = call(x, t, 2, torch.tensor(rows, dtype=torch.int32, device=DEV))
        check_peaked(got, [pairs[r][2] for r in rows], leads)
        assert got[3].tolist() == [[pairs[r][0], pairs[r][1]] for r in rows]


@pytest.mark.gpu
@pytest.mark.parametrize("n", [32, 20000])
@pytest.mark.parametrize("cap", [5.0, 30.0])
def test_capped_logits_by_themselves(n, cap):
    """A vocabulary of one id: ln sum exp is the capped logit, with no rounding beside it.  From 1/4 of a cap on: the exponential's argument is 2 z log2(e) with
    z, the constant and the product rounded (4 times 2^-24 of it), tanh falls by z sech^2 z <= 0.45 of that; the exponential (2^-22 of itself, times at most 0.47 = 2 e / (e + 1)^2), the
    reciprocal (2^-23, times 0.76) and two roundings come to 1.8 times 2^-22 of the cap with it; below 1/4 three or four roundings of the series, of up to 1/4 of the cap."""
    w = torch.zeros(1, 8, device=DEV, dtype=torch.bfloat16)
    w[0, 0] = 1.0
    g = torch.Generator(device=DEV).manual_seed(n)
    for scale in (1.0, 1.01171875, 0.1):
        h = torch.zeros(n, 8, device=DEV, dtype=torch.bfloat16)
        h[:, 0] = ((torch.rand(n, generator=g, device=DEV) * 2 - 1) * 4 * cap).to(torch.bfloat16)
        got = head(h, w, torch.zeros(n, dtype=torch.int32, device=DEV), 0, scale, cap)
        z = (h[:, 0].float() * torch.tensor(scale, device=DEV)).double().cpu() / cap
        assert float((got[2].double() - cap * torch.tanh(z)).abs().max()) <= cap * 1.8 * 2.0 ** -22
        assert bool((got[0] == 0).all()) and bool((got[1] == 0).all())
