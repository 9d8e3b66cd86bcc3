"""Ragged prefill attention over the 8-bit cache against the 64-bit definition."""
import numpy as np
import pytest
import torch

import kv8_reference as ref
from kv8_reference import E4M3, INT8
from test_kv8_gpu import BF16_HALF_STEP, bf16, check_decode, dev, gpu_cache, laid_out, refused, unit_of, values_of

pytestmark = pytest.mark.gpu

# A rounding to binary16 is off by at most half a step, 2^-11 of the value.  There are three on a
# key's way: its weight, its V scale relative to the largest (exact for powers of two, which these
# caches do not have) and that scale times the code.  Together 3 * 2^-11 of p |v|.  Below binary16's
# normal range a rounding is off by 2^-25: of a weight where the row's largest is at least 1, and of
# a V value where 64 times the largest code is the largest; at most 2^-24 of `unit` per key.
WEIGHT_AND_V = 3 * 2.0 ** -11


def check_prefill(gpu, code, shape, seqs, bt, seed=0, q_scale=1.0, scale=0.0, softcap=0.0, window=0, slopes=None,
                  prefix=None, drop=(), levels=(-9, -4), pad=0, max_rows=None, max_ctx=None, q=None, strided=False,
                  workspace=None):
    """seqs: (rows, context) of each sequence."""
    q_heads, heads, dim = shape
    rng = np.random.default_rng(seed)
    lens = [c for _, c in seqs]
    codes, scales, tables = laid_out(rng, code, lens, heads, bt, dim, levels)
    whole = tables.copy()
    for page, bad in drop:
        if page < tables.shape[1]:
            tables[:, page] = bad
    starts = np.concatenate(([0], np.cumsum([r for r, _ in seqs]))).astype(np.int32)
    n_rows = int(starts[-1]) + pad
    if q is None:
        q = rng.standard_normal((n_rows, q_heads, dim)) * q_scale
    q = bf16(q)
    dq = dev(q, torch.bfloat16)
    if strided:
        wide = torch.zeros(n_rows, q_heads * dim + 64, dtype=torch.bfloat16, device="cuda")
        wide[:, 32:32 + q_heads * dim] = dq.view(n_rows, -1)
        dq = wide[:, 32:32 + q_heads * dim].view(n_rows, q_heads, dim)
    out = torch.full((n_rows, q_heads, dim), -7.0, dtype=torch.bfloat16, device="cuda")
    cache = gpu_cache(gpu, codes, scales, code)
    options = gpu.ScoreOptions(scale, softcap, window, None if slopes is None else dev(slopes, torch.float32),
                               None if prefix is None else dev(np.asarray(prefix, np.int32)))
    ws = gpu.kv8_prefill_bf16(cache, dq, dev(tables), dev(np.asarray(lens, np.int32)), dev(starts), out,
                              max_rows=max_rows, max_ctx=max_ctx, options=options, workspace=workspace)
    got = out.double().cpu().numpy()
    if ws is not None:
        assert not ws[:16384].any()
    assert (got[starts[-1]:] == -7.0).all()
    slopes64 = None if slopes is None else np.asarray(slopes, np.float32).astype(np.float64)
    for b, (r, c) in enumerate(seqs):
        at = slice(starts[b], starts[b + 1])
        if r == 0:
            continue
        if c <= 0:
            assert not got[at].any()
            continue
        present = np.ones(c, bool)
        for page, _ in drop:
            present[page * bt:(page + 1) * bt] = False
        k, v = values_of(codes, scales, code, whole[b], c, bt)
        want, bound = ref.attention(q[at], k, v, np.arange(c - r, c), scale, softcap, window, slopes64,
                                    prefix=0 if prefix is None else prefix[b], present=present,
                                    unit=unit_of(scales, code) * 2.0 ** 15)
        spread, _ = ref.attention(q[at], k, np.abs(v), np.arange(c - r, c), scale, softcap, window, slopes64,
                                  prefix=0 if prefix is None else prefix[b], present=present)
        # sum p |v| carries the weights' and V's own roundings, and those of the sum of weights
        bound = bound + spread * WEIGHT_AND_V + np.abs(want) * BF16_HALF_STEP + 2.0 ** -133
        if softcap > 0:  # 1 - 2 / (e^2x + 1) in f32: 2^-22 of the cap, in a score
            bound = bound + 2 * spread * softcap * 1.5 * 2.0 ** -22
        err = np.abs(got[at] - want)
        assert (err <= bound).all(), (b, r, c, float((err / bound).max()), float(err.max()))
    return out


SHAPES = [(32, 4, 64), (32, 8, 128), (12, 12, 64), (8, 2, 128), (5, 1, 64), (21, 3, 128)]


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("seqs,bt", [
    ([(1, 1)], 16), ([(64, 64)], 16), ([(65, 65), (1, 130), (33, 200)], 32), ([(130, 130)], 256),
    ([(2, 700), (0, 40), (17, 17), (100, 399)], 64)])
def test_prefill(gpu, code, shape, seqs, bt):
    check_prefill(gpu, code, shape, seqs, bt)


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("options", [
    dict(softcap=30.0), dict(softcap=0.5, q_scale=30.0), dict(slopes=True), dict(slopes=True, softcap=20.0),
    dict(window=1), dict(window=64), dict(window=100, slopes=True), dict(window=2 ** 31 - 1), dict(scale=0.37),
    dict(prefix=[70, 0, 300, 5]), dict(prefix=[200, 1000, 64, 1], window=40), dict(prefix=[70, 30, 300, 5], slopes=True)])
def test_prefill_options(gpu, code, options):
    o = dict(options)
    if o.get("slopes"):
        o["slopes"] = 2.0 ** (-8.0 * np.arange(1, 9) / 8)
    check_prefill(gpu, code, (8, 2, 64), [(70, 200), (64, 64), (30, 300), (1, 5)], 16, **o)
    check_prefill(gpu, code, (8, 4, 128), [(70, 200), (64, 64), (30, 300), (1, 5)], 32, **o)


# Few rows per sequence: launches whose (row, head) pairs the decode's kernel takes.
FEW = [(4, 200), (3, 3), (1, 300), (0, 50), (4, 64), (2, 1000), (4, 5)]


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("shape,most", [((16, 4, 128), 4), ((8, 2, 64), 4), ((5, 1, 64), 3), ((21, 3, 128), 2),
                                        ((4, 4, 64), 4), ((32, 2, 64), 4), ((15, 1, 128), 4), ((17, 1, 64), 1)])
def test_prefill_of_few_rows(gpu, code, shape, most):
    seqs = [(min(r, most), c) for r, c in FEW]
    check_prefill(gpu, code, shape, seqs, 16)
    check_prefill(gpu, code, shape, seqs, 64, strided=True, pad=len(seqs) * most - sum(r for r, _ in seqs),
                  max_rows=most)
    check_prefill(gpu, code, shape, [(most, 4000)], 32)


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("options", [
    dict(softcap=30.0), dict(softcap=0.5, q_scale=30.0), dict(slopes=True), dict(slopes=True, softcap=20.0),
    dict(window=1), dict(window=3), dict(window=64), dict(window=100, slopes=True), dict(window=2 ** 31 - 1),
    dict(scale=0.37), dict(prefix=[70, 0, 300, 5, 64, 998, 9]), dict(prefix=[200, 1000, 64, 1, 61, 0, 3], window=40),
    dict(prefix=[199, 30, 300, 5, 62, 500, 4], slopes=True), dict(drop=[(0, -1), (2, 1 << 20)])])
def test_prefill_of_few_rows_options(gpu, code, options):
    o = dict(options)
    if o.get("slopes"):
        o["slopes"] = 2.0 ** (-8.0 * np.arange(1, 9) / 8)
    check_prefill(gpu, code, (8, 2, 64), FEW, 16, **o)      # 16 pairs
    check_prefill(gpu, code, (8, 1, 128), FEW, 32, **o)     # 32


def test_prefill_of_few_rows_of_many_sequences(gpu):
    rng = np.random.default_rng(70)
    for n, shape in ((70, (8, 2, 64)), (1100, (2, 1, 64))):
        check_prefill(gpu, E4M3, shape, [(int(r), int(r + c)) for r, c in zip(rng.integers(0, 5, n), rng.integers(0, 90, n))],
                      16, max_rows=4)


def test_prefill_of_few_rows_keeps_nan_to_its_row(gpu):
    rng = np.random.default_rng(71)
    codes, scales, tables = laid_out(rng, E4M3, [700], 2, 16, 64)
    cache, q = gpu_cache(gpu, codes, scales, E4M3), torch.randn(4, 8, 64, device="cuda").bfloat16()
    call = lambda q: gpu.kv8_prefill_bf16(cache, q, dev(tables), dev(np.array([700], np.int32)),  # noqa: E731
                                          dev(np.array([0, 4], np.int32)), out)
    out = torch.empty_like(q)
    call(q)
    want = out.clone()
    q[1, 3, 5], q[2, 6, 0] = float("nan"), float("inf")
    call(q)
    assert out[1, 3].isnan().all() and out[2, 6].isnan().all()
    out[1, 3], out[2, 6] = want[1, 3], want[2, 6]
    assert torch.equal(out, want)


@pytest.mark.parametrize("code,softcap", [(E4M3, 0.0), (INT8, 20.0)])
@pytest.mark.parametrize("shape", [(2, 1, 64), (2, 2, 128)])
def test_prefill_of_biased_rows_within_prefixes(gpu, code, softcap, shape):
    """Keys in front of a wavefront's rows, around them and behind all of them."""
    slopes = 2.0 ** (-8.0 * np.arange(1, 3) / 2)
    check_prefill(gpu, code, shape, [(300, 420), (90, 400), (64, 640)], 16, slopes=slopes, softcap=softcap,
                  prefix=[400, 390, 640])


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("options", [
    dict(), dict(softcap=30.0), dict(slopes=True), dict(slopes=True, softcap=20.0, window=100),
    dict(slopes=True, prefix=True), dict(drop=[(1, -1)])])
def test_prefill_of_many_tiles(gpu, code, options):
    """Launches that workgroups of eight wavefronts take, in whole tiles and with ragged ends."""
    rng = np.random.default_rng(12)
    rows = [32] * 30 + [33, 1, 31, 60, 35] + [32] * 29
    o = dict(options)
    if o.get("slopes"):
        o["slopes"] = 2.0 ** (-8.0 * np.arange(1, 65) / 64)
    if o.get("prefix"):
        o["prefix"] = rng.integers(0, 150, len(rows)).tolist()
    check_prefill(gpu, code, (64, 8, 128), [(r, r + int(n)) for r, n in zip(rows, rng.integers(0, 150, len(rows)))], 16, **o)


@pytest.mark.parametrize("shape", [(32, 4, 64), (8, 2, 128)])
@pytest.mark.parametrize("seqs", [[(3, 5000)], [(40, 9000)], [(1, 3000), (16, 2000), (1, 1)], [(300, 8500)]])
def test_prefill_with_the_keys_cut_into_pieces(gpu, shape, seqs):
    check_prefill(gpu, E4M3, shape, seqs, 16)


def test_prefill_of_a_padded_batch(gpu):
    """Rows behind the last sequence stay as they were; empty contexts, and rows at negative positions."""
    check_prefill(gpu, E4M3, (8, 2, 64), [(0, 0), (5, 40), (4, 0), (0, 9), (9, 9)], 16, pad=77)
    check_prefill(gpu, E4M3, (8, 2, 64), [(10, 6), (3, 3)], 16, pad=1)


def test_prefill_of_more_sequences_than_a_launch_takes(gpu):
    rng = np.random.default_rng(3)
    check_prefill(gpu, INT8, (4, 2, 64), [(int(r), int(r + h)) for r, h in rng.integers(0, 20, (1100, 2))], 16, pad=3)


def test_prefill_does_not_depend_on_its_bounds(gpu):
    for max_rows, max_ctx in ((1, 1), (100, 100), (5000, 100000)):
        check_prefill(gpu, E4M3, (8, 2, 64), [(90, 1900), (33, 33)], 16, max_rows=max_rows, max_ctx=max_ctx)


@pytest.mark.parametrize("held", [1, 31, 32, 70, 71])
def test_prefill_of_fewer_rows_than_the_starts_tell(gpu, held):
    """Positions go by row_starts: the rows that q holds are those of the whole batch."""
    rng = np.random.default_rng(40)
    lens = [90, 200, 64]
    codes, scales, tables = laid_out(rng, E4M3, lens, 2, 16, 64)
    cache, q = gpu_cache(gpu, codes, scales, E4M3), torch.randn(102, 8, 64, device="cuda").bfloat16()
    starts, dlens = dev(np.array([0, 31, 71, 102], np.int32)), dev(np.asarray(lens, np.int32))
    whole, part = torch.empty_like(q), torch.full_like(q, -7.0)
    gpu.kv8_prefill_bf16(cache, q, dev(tables), dlens, starts, whole)
    gpu.kv8_prefill_bf16(cache, q[:held], dev(tables), dlens, starts, part[:held])
    assert torch.equal(part[:held], whole[:held]) and (part[held:] == -7.0).all()


def test_prefill_skips_pages_that_are_no_blocks(gpu):
    for drop in ([(1, -1)], [(0, 2 ** 31 - 1), (5, -7)], [(4, 10 ** 6), (5, -1), (6, -1), (7, -1)],
                 [(i, -1) for i in range(100)]):
        check_prefill(gpu, E4M3, (8, 2, 64), [(60, 160), (97, 97), (16, 16)], 16, drop=drop)


def test_prefill_of_scales_far_apart(gpu):
    check_prefill(gpu, E4M3, (8, 2, 64), [(60, 300)], 16, levels=(-9, 0), q_scale=0.5)
    check_prefill(gpu, INT8, (8, 2, 64), [(60, 300)], 16, levels=(-60, -50))
    check_prefill(gpu, INT8, (8, 2, 64), [(60, 300)], 16, levels=(30, 40), q_scale=1e-11)


def test_prefill_of_extreme_q(gpu):
    rng = np.random.default_rng(4)
    q = rng.standard_normal((60, 8, 64)) * np.exp(2 * rng.standard_normal((60, 8, 64)))
    check_prefill(gpu, E4M3, (8, 2, 64), [(60, 200)], 16, q=q * 1e6, scale=1e-7)
    check_prefill(gpu, E4M3, (8, 2, 64), [(60, 200)], 16, q=q * 1e-36, scale=1e35)
    check_prefill(gpu, E4M3, (8, 2, 64), [(60, 200)], 16, q=q * 0)


def test_prefill_of_long_ranges(gpu):
    """More keys than one table of pages holds."""
    check_prefill(gpu, E4M3, (1, 1, 64), [(2, 17000)], 16, max_ctx=64)
    check_prefill(gpu, E4M3, (1, 1, 128), [(70, 8400)], 64, max_ctx=64)


def test_prefill_of_long_ranges_in_many_tiles(gpu):
    """The same by workgroups of eight wavefronts: sequences that share their pages, of many heads, three of which
    are compared."""
    rng = np.random.default_rng(50)
    heads, ctx, rows = 64, 8400, [129, 150, 130, 256, 140, 200, 129, 180]
    codes, scales, tables = laid_out(rng, E4M3, [ctx], heads, 64, 128)
    starts = np.concatenate(([0], np.cumsum(rows))).astype(np.int32)
    q = torch.randn(int(starts[-1]), heads, 128, device="cuda").bfloat16()
    out = torch.empty_like(q)
    lens = np.array([ctx - 30 * b for b in range(len(rows))], np.int32)
    gpu.kv8_prefill_bf16(gpu_cache(gpu, codes, scales, E4M3), q, dev(np.repeat(tables, len(rows), 0)), dev(lens),
                         dev(starts), out)
    for b, h in ((0, 0), (3, 17), (7, 63)):
        at, n = slice(starts[b], starts[b + 1]), int(lens[b])
        k, v = values_of(codes[:, :, h:h + 1], scales[:, :, h:h + 1], E4M3, tables[0], n, 64)
        qh, pos = q[at, h:h + 1].double().cpu().numpy(), n - rows[b] + np.arange(rows[b])
        want, bound = ref.attention(qh, k, v, pos, unit=unit_of(scales[:, :, h:h + 1], E4M3) * 2.0 ** 15)
        spread, _ = ref.attention(qh, k, np.abs(v), pos)
        err = np.abs(out[at, h:h + 1].double().cpu().numpy() - want)
        assert (err <= bound + spread * WEIGHT_AND_V + np.abs(want) * BF16_HALF_STEP + 2.0 ** -133).all()


def test_prefill_of_rows_of_a_wider_projection(gpu):
    check_prefill(gpu, E4M3, (8, 2, 64), [(60, 160), (3, 3)], 16, strided=True)


def test_prefill_keeps_nan_to_its_row(gpu):
    rng = np.random.default_rng(6)
    codes, scales, tables = laid_out(rng, E4M3, [300], 2, 16, 64)
    cache, q = gpu_cache(gpu, codes, scales, E4M3), torch.randn(70, 8, 64, device="cuda").bfloat16()
    lens, starts, tables = dev(np.array([300], np.int32)), dev(np.array([0, 70], np.int32)), dev(tables)
    clean, out = torch.empty_like(q), torch.empty_like(q)
    gpu.kv8_prefill_bf16(cache, q, tables, lens, starts, clean)
    q[9, 3, 5], q[69, 6, 1] = float("nan"), float("inf")
    gpu.kv8_prefill_bf16(cache, q, tables, lens, starts, out)
    assert out[9, 3].isnan().all() and out[69, 6].isnan().all()
    out[9, 3], out[69, 6] = clean[9, 3], clean[69, 6]
    assert torch.equal(out, clean)


def test_prefill_of_one_row_is_decode(gpu):
    rng = np.random.default_rng(16)
    lens = [500, 33, 1, 64]
    codes, scales, tables = laid_out(rng, E4M3, lens, 2, 16, 128)
    cache, q = gpu_cache(gpu, codes, scales, E4M3), torch.randn(4, 8, 128, device="cuda").bfloat16()
    dlens, tables = dev(np.asarray(lens, np.int32)), dev(tables)
    a, b = torch.empty_like(q), torch.empty_like(q)
    gpu.kv8_decode(cache, q, tables, dlens, a)
    gpu.kv8_prefill_bf16(cache, q, tables, dlens, dev(np.arange(5, dtype=np.int32)), b)
    # each is within its own bound; bf16's steps are the largest part
    assert ((a.float() - b.float()).abs() <= a.float().abs() * 2.0 ** -7 + a.float().abs().amax() * 2.0 ** -8).all()


def test_calls_of_many_shapes_take_turns_in_one_workspace(gpu):
    ws = torch.full((1 << 26,), 0xff, dtype=torch.uint8, device="cuda")  # only the counters' part starts at zero
    ws[:16384] = 0
    for i in range(2):
        check_decode(gpu, E4M3, [4000 - 900 * i], 16, 2, 16, 64, workspace=ws)
        check_decode(gpu, INT8, [700, 1, 0, 300 + i] * 24, 8, 8, 32, 128, workspace=ws)
        check_prefill(gpu, E4M3, (8, 2, 64), [(64, 3000)], 32, workspace=ws)
        check_decode(gpu, E4M3, list(range(1, 2000, 40)), 4, 4, 16, 64, workspace=ws)
        check_prefill(gpu, INT8, (4, 1, 128), [(33, 1500), (0, 40), (5, 900 + i)], 16, workspace=ws)
        check_decode(gpu, E4M3, [2500, 900], 32, 1, 64, 128, io="bf16", workspace=ws)
        check_prefill(gpu, E4M3, (8, 2, 64), [(2, 2900 + i), (1, 40), (4, 1000)], 32, workspace=ws)
    assert not ws[:16384].any()


def test_prefill_in_graphs(gpu):
    """Captured once with its bounds, replayed with other lengths between eager calls."""
    rng = np.random.default_rng(7)
    seqs = [(30, 3000), (1, 500), (64, 900)]
    codes, scales, tables = laid_out(rng, E4M3, [c for _, c in seqs], 2, 16, 64)
    cache, q = gpu_cache(gpu, codes, scales, E4M3), torch.randn(95, 8, 64, device="cuda").bfloat16()
    dlens = dev(np.array([c for _, c in seqs], np.int32))
    starts, tables = dev(np.array([0, 30, 31, 95], np.int32)), dev(tables)
    outs = [torch.zeros_like(q) for _ in range(2)]
    ws = [gpu.alloc_workspace(gpu.kv8_prefill_workspace_size(cache, 3, 8, 95, 64, 3000)) for _ in range(2)]
    graphs, side = [], torch.cuda.Stream()
    for o, w in zip(outs, ws):
        g = torch.cuda.CUDAGraph()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(g, stream=side):
            gpu.kv8_prefill_bf16(cache, q, tables, dlens, starts, o, max_rows=64, max_ctx=3000, workspace=w)
        graphs.append(g)
    torch.cuda.synchronize()
    for step in range(4):
        dlens.copy_(torch.tensor([3000 - 700 * step, 500, 900 - 13 * step], dtype=torch.int32))
        starts.copy_(torch.tensor([0, 30 - 7 * step, 31 - 6 * step, 95 - 8 * step], dtype=torch.int32))
        q.copy_(torch.randn(95, 8, 64).bfloat16())
        eager = torch.zeros_like(q)
        gpu.kv8_prefill_bf16(cache, q, tables, dlens, starts, eager, max_rows=64, max_ctx=3000)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert eager.isfinite().all()
        assert torch.equal(outs[0], eager) and torch.equal(outs[1], eager), step
        for o in outs:
            o.zero_()


def test_a_captured_step_serves_other_batches(gpu):
    """Map, write and attention captured once, for at most five sequences and 96 rows, replayed for batches of other
    lengths, padded ones among them, against the same calls made eagerly."""
    heads, q_heads, bt, dim, batch, n_rows, n_blocks = 2, 8, 16, 64, 5, 96, 64
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731

    def state():
        return dict(cache=gpu.Kv8Cache.empty(n_blocks, heads, bt, dim), cached=i32(batch), new=i32(batch),
                    free=i32(n_blocks), tables=torch.full((batch, 20), -1, dtype=torch.int32, device="cuda"),
                    ctx=i32(batch), starts=i32(batch + 1), slots=torch.zeros(n_rows, dtype=torch.int64, device="cuda"),
                    positions=i32(n_rows), counts=i32(2), kv=torch.zeros(2, n_rows, heads, dim, device="cuda"),
                    q=torch.zeros(n_rows, q_heads, dim, dtype=torch.bfloat16, device="cuda"),
                    out=torch.zeros(n_rows, q_heads, dim, dtype=torch.bfloat16, device="cuda"),
                    ws=gpu.alloc_workspace(1 << 24))

    def step(s):
        gpu.batch_map(s["cached"], s["new"], s["free"], s["tables"], bt, n_blocks, s["ctx"], s["starts"], s["slots"],
                      s["positions"], s["counts"])
        gpu.kv8_write(s["cache"], s["slots"], s["kv"][0], s["kv"][1])
        gpu.kv8_prefill_bf16(s["cache"], s["q"], s["tables"], s["ctx"], s["starts"], s["out"], max_rows=90, max_ctx=300,
                             workspace=s["ws"])

    eager, graphed = state(), state()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(graphed)
    rng, lens, left = np.random.default_rng(61), np.zeros(batch, np.int32), rng_blocks(n_blocks)
    for new in ([40, 3, 0, 17, 0], [1, 1, 0, 1, 0], [1, 16, 60, 1, 1], [0, 0, 0, 0, 0], [90, 1, 1, 1, 3], [1, 1, 1, 1, 1]):
        new = np.array(new, np.int32)
        kv = torch.from_numpy(rng.standard_normal((2, n_rows, heads, dim)).astype(np.float32)).cuda()
        q = torch.from_numpy(rng.standard_normal((n_rows, q_heads, dim)).astype(np.float32)).cuda().bfloat16()
        for s in (eager, graphed):
            s["cached"].copy_(dev(lens)), s["new"].copy_(dev(new)), s["kv"].copy_(kv), s["q"].copy_(q)
            s["free"].fill_(-1)
            s["free"][:len(left)].copy_(dev(left)), s["out"].fill_(-7.0)
        step(eager)
        graph.replay()
        torch.cuda.synchronize()
        for name in ("tables", "ctx", "starts", "slots", "positions", "counts", "out"):
            assert torch.equal(eager[name], graphed[name]), name
        for name in ("k", "v", "k_scales", "v_scales"):
            assert torch.equal(getattr(eager["cache"], name), getattr(graphed["cache"], name)), name
        lens, rows = lens + new, int(new.sum())
        assert (eager["ctx"].cpu().numpy() == lens).all() and int(eager["counts"][1]) == rows
        assert (eager["out"][rows:] == -7.0).all() and eager["out"][:rows].isfinite().all()
        left = left[int(eager["counts"][0]):]


def test_prefill_of_few_rows_in_graphs(gpu):
    rng = np.random.default_rng(72)
    codes, scales, tables = laid_out(rng, E4M3, [3000, 500, 900], 2, 16, 64)
    cache, q = gpu_cache(gpu, codes, scales, E4M3), torch.randn(12, 8, 64, device="cuda").bfloat16()
    dlens, starts = dev(np.array([3000, 500, 900], np.int32)), dev(np.array([0, 4, 5, 9], np.int32))
    tables, out, eager = dev(tables), torch.zeros_like(q), torch.zeros_like(q)
    ws, graph = gpu.alloc_workspace(gpu.kv8_prefill_workspace_size(cache, 3, 8, 12, 4, 3000)), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu.kv8_prefill_bf16(cache, q, tables, dlens, starts, out, max_rows=4, max_ctx=3000, workspace=ws)
    for step, rows in enumerate(([4, 1, 4], [4, 4, 4], [0, 2, 3], [1, 1, 1])):
        dlens.copy_(torch.tensor([3000 - 700 * step, 500 - step, 900 - 13 * step], dtype=torch.int32))
        starts.copy_(dev(np.concatenate(([0], np.cumsum(rows))).astype(np.int32)))
        q.copy_(torch.randn(12, 8, 64).bfloat16())
        out.fill_(-7.0), eager.fill_(-7.0)
        gpu.kv8_prefill_bf16(cache, q, tables, dlens, starts, eager, max_rows=4, max_ctx=3000)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and eager.isfinite().all(), step
        assert (out[sum(rows):] == -7.0).all() and not (out[:sum(rows)] == -7.0).all()


def rng_blocks(n):
    return np.random.default_rng(n).permutation(n).astype(np.int32)


def test_prompts_then_decode(gpu):
    """A batch's prompts mapped, written and attended in one step, then a decode step on top of them."""
    rng = np.random.default_rng(31)
    heads, q_heads, bt, dim, batch = 2, 8, 32, 128, 4
    cache = gpu.Kv8Cache.empty(40, heads, bt, dim)
    tables = torch.full((batch, 10), -1, dtype=torch.int32, device="cuda")
    free = dev(rng.permutation(40).astype(np.int32))
    codes, scales = np.zeros((2, 40, heads, bt, dim), np.uint8), np.zeros((2, 40, heads))
    lens = torch.zeros(batch, dtype=torch.int32, device="cuda")
    for new in ([70, 1, 128, 33], [9, 40, 1, 64], [1, 1, 1, 1]):
        n_rows = sum(new) + 6
        i32 = lambda *s: torch.empty(*s, dtype=torch.int32, device="cuda")  # noqa: E731
        ctx, starts, counts, positions = i32(batch), i32(batch + 1), i32(2), i32(n_rows)
        slots = torch.empty(n_rows, dtype=torch.int64, device="cuda")
        gpu.batch_map(lens, dev(np.asarray(new, np.int32)), free, tables, bt, 40, ctx, starts, slots, positions, counts)
        x = bf16(rng.standard_normal((2, n_rows, heads, dim)))
        gpu.kv8_write(cache, slots, dev(x[0], torch.bfloat16), dev(x[1], torch.bfloat16))
        q = bf16(rng.standard_normal((n_rows, q_heads, dim)))
        dq, out = dev(q, torch.bfloat16), torch.zeros(n_rows, q_heads, dim, dtype=torch.bfloat16, device="cuda")
        if max(new) == 1:
            gpu.kv8_decode(cache, dq[:batch], tables, ctx, out[:batch])
        else:
            gpu.kv8_prefill_bf16(cache, dq, tables, ctx, starts, out, max_rows=128, max_ctx=300)
        free, lens = free[int(counts[0]):], ctx
        for i in range(2):
            ref.write(codes[i], scales[i], slots.cpu().numpy(), x[i], E4M3)
        got, table = out.double().cpu().numpy(), tables.cpu().numpy()
        assert not got[sum(new):].any()
        for b, c in enumerate(ctx.tolist()):
            at = slice(int(starts[b]), int(starts[b + 1]))
            k, v = values_of(codes, scales, E4M3, table[b], c, bt)
            pos = np.arange(c - new[b], c)
            want, bound = ref.attention(q[at], k, v, pos, unit=unit_of(scales, E4M3) * 2.0 ** 15)
            spread, _ = ref.attention(q[at], k, np.abs(v), pos)
            bound = bound + spread * WEIGHT_AND_V + np.abs(want) * BF16_HALF_STEP
            assert (np.abs(got[at] - want) <= bound).all()


def test_prefill_refusals(gpu):
    cache = gpu.Kv8Cache.empty(8, 2, 16, 64)
    q = torch.zeros(6, 8, 64, dtype=torch.bfloat16, device="cuda")
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    call = lambda **k: gpu.kv8_prefill_bf16(**{**dict(  # noqa: E731
        cache=cache, q=q, block_tables=i32(2, 400), ctx_lens=i32(2), row_starts=i32(3), out=torch.empty_like(q),
        max_rows=6, max_ctx=6000), **k})
    INV, WS = gpu.ERR_INVALID, gpu.ERR_WORKSPACE
    refused(gpu, WS, lambda: call(workspace=torch.zeros(256, dtype=torch.uint8, device="cuda")))
    refused(gpu, INV, lambda: call(workspace=gpu.alloc_workspace(1 << 26)[8:]))
    refused(gpu, INV, lambda: call(q=q.float(), out=torch.empty_like(q).float()))
    refused(gpu, INV, lambda: call(q=q[:, :7]))
    refused(gpu, INV, lambda: call(row_starts=i32(2)))
    refused(gpu, INV, lambda: call(row_starts=i32(3).cpu()))
    refused(gpu, INV, lambda: call(max_rows=0))
    refused(gpu, INV, lambda: call(max_ctx=-1))
    refused(gpu, INV, lambda: call(options=gpu.ScoreOptions(prefix_lens=i32(3))))
    refused(gpu, INV, lambda: call(options=gpu.ScoreOptions(softcap=float("inf"))))
    call(q=q[:0], out=torch.empty_like(q)[:0])  # no rows: nothing to do
