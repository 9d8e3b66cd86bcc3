"""Batched serving on the 8-bit cache: the batch map, the write and decode attention against the
64-bit definitions, and a run of them together."""
import numpy as np
import pytest
import torch

import kv8_reference as ref
from kv8_reference import E4M3, INT8

pytestmark = pytest.mark.gpu

BF16_HALF_STEP = 2.0 ** -8


def dev(x, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x))
    return t.cuda() if dtype is None else t.to(dtype).cuda()


def bf16(x):
    """x rounded to bf16, as float64."""
    return torch.from_numpy(np.asarray(x, np.float32)).bfloat16().double().numpy()


# ------------------------------------------------------------- batch map

def run_map(gpu, cached, new, free, tables, bt, num_blocks, n_rows):
    B = len(cached)
    t = dev(tables)
    out = dict(ctx_lens=torch.full((B,), -7, dtype=torch.int32, device="cuda"),
               row_starts=torch.full((B + 1,), -7, dtype=torch.int32, device="cuda"),
               slots=torch.full((n_rows,), -7, dtype=torch.int64, device="cuda"),
               positions=torch.full((n_rows,), -7, dtype=torch.int32, device="cuda"),
               counts=torch.full((2,), -7, dtype=torch.int32, device="cuda"))
    gpu.batch_map(dev(np.asarray(cached, np.int32)), dev(np.asarray(new, np.int32)),
                  dev(np.asarray(free, np.int32)), t, bt, num_blocks, **out)
    return t.cpu().numpy(), {k: x.cpu().numpy() for k, x in out.items()}


@pytest.mark.parametrize("batch,bt,cached_hi,new_hi,free_share,pad,pages", [
    (1, 16, 0, 1, 2.0, 0, 4), (1, 16, 40, 300, 2.0, 5, 40), (64, 16, 500, 1, 2.0, 0, 40),
    (64, 16, 500, 0, 2.0, 3, 40), (63, 32, 100, 70, 0.5, 11, 8), (513, 64, 900, 5, 2.0, 0, 16),
    (1025, 16, 60, 40, 0.9, 1000, 5), (7, 256, 1000, 3000, 2.0, 0, 20), (4096, 16, 20, 3, 2.0, 1, 3),
    (3, 1, 5, 9, 2.0, 0, 30)])
def test_map(gpu, batch, bt, cached_hi, new_hi, free_share, pad, pages):
    rng = np.random.default_rng(batch * 31 + bt)
    cached = rng.integers(0, cached_hi + 1, batch)
    new = rng.integers(0, new_hi + 1, batch)
    if new_hi == 1:
        new[:] = 1
    held = -(-cached // bt)
    tables = np.full((batch, pages), -5, np.int32)
    order = rng.permutation(held.sum() + 100000).astype(np.int32)
    at = 0
    for b in range(batch):
        n = min(held[b], pages)
        tables[b, :n] = order[at:at + n]
        at += n
    wanted = int((-(-(cached + new) // bt) - held).sum())
    free = order[at:at + int(wanted * free_share)]
    num_blocks = len(order) - 1000  # some ids are not blocks of the cache
    n_rows = int(new.sum()) + pad
    want_t = tables.copy()
    want = ref.batch_map(cached, new, free, want_t, bt, num_blocks, n_rows)
    got_t, got = run_map(gpu, cached, new, free, tables, bt, num_blocks, n_rows)
    assert np.array_equal(got_t, want_t)
    for name, w in zip(("ctx_lens", "row_starts", "slots", "positions", "counts"), want):
        assert np.array_equal(got[name], w), name


def test_map_of_more_rows_than_the_outputs_hold(gpu):
    cached, new = np.array([3, 0, 17]), np.array([20, 9, 30])
    tables = np.zeros((3, 8), np.int32)
    free = np.arange(10, 20, dtype=np.int32)
    want_t = tables.copy()
    want = ref.batch_map(cached, new, free, want_t, 16, 64, 33)
    got_t, got = run_map(gpu, cached, new, free, tables, 16, 64, 33)
    assert np.array_equal(got_t, want_t) and np.array_equal(got["slots"], want[2])
    assert np.array_equal(got["row_starts"], want[1]) and got["counts"][1] == 59


def test_map_of_negative_and_huge_lengths(gpu):
    """Negative lengths count as 0; sums that leave 32 bits stop at 2^31 - 1 and write nothing wrong."""
    big = 2 ** 31 - 1
    cached, new = np.array([-4, big - 2, 5]), np.array([2, big, -3])
    tables = np.zeros((3, 2), np.int32)
    got_t, got = run_map(gpu, cached, new, np.arange(1, 9), tables, 16, 64, 40)
    assert got["ctx_lens"].tolist() == [2, big, 5]
    assert got["row_starts"].tolist() == [0, 2, big, big]
    assert got["slots"][:2].tolist() == [16, 17] and (got["slots"][2:] == -1).all()
    assert got_t.tolist() == [[1, 0], [0, 0], [0, 0]] and got["counts"].tolist() == [1, big]


# ------------------------------------------------------------- write

def random_cache(rng, code, blocks, heads, bt, dim):
    """Finite codes and positive scales (powers of two), for K and V."""
    codes = rng.integers(0, 256, (2, blocks, heads, bt, dim)).astype(np.uint8)
    if code == E4M3:
        codes[(codes & 127) == 127] = 0x35
    else:
        codes[codes == 128] = 3
    scales = 2.0 ** rng.integers(-9, -4, (2, blocks, heads))
    return codes, scales.astype(np.float32)


def gpu_cache(gpu, codes, scales, code):
    return gpu.Kv8Cache(dev(codes[0]), dev(codes[1]), dev(scales[0]), dev(scales[1]), code)


def check_cache(cache, codes, scales):
    for got, want in ((cache.k, codes[0]), (cache.v, codes[1])):
        diff = got.cpu().numpy() != want
        # +0 and -0 are one value
        got, want = got.cpu().numpy(), want
        if cache.code == E4M3:
            diff &= ~(((got & 127) == 0) & ((want & 127) == 0))
        assert not diff.any(), (int(diff.sum()), np.argwhere(diff)[:4])
    assert np.array_equal(cache.k_scales.cpu().numpy(), scales[0].astype(np.float32))
    assert np.array_equal(cache.v_scales.cpu().numpy(), scales[1].astype(np.float32))


def run_write(gpu, code, blocks, heads, bt, dim, slots, x, io, seed=0, stride=None):
    """Writes x [2][rows][heads][dim] and compares every code and scale with the definition."""
    rng = np.random.default_rng(seed)
    codes, scales = random_cache(rng, code, blocks, heads, bt, dim)
    cache = gpu_cache(gpu, codes, scales, code)
    x = np.asarray(x, np.float32)
    if io == "bf16":
        x = bf16(x).astype(np.float32)
    t = [dev(x[i], torch.bfloat16 if io == "bf16" else torch.float32) for i in range(2)]
    if stride:  # rows of a wider projection
        wide = [torch.full((x.shape[1], stride), float("nan"), dtype=u.dtype, device="cuda") for u in t]
        for u, w in zip(t, wide):
            w[:, 16:16 + heads * dim] = u.view(len(u), -1)
        t = [w[:, 16:16 + heads * dim].view(-1, heads, dim) for w in wide]
    gpu.kv8_write(cache, dev(np.asarray(slots, np.int64)), *t)
    ks, want = scales.astype(np.float64), codes.copy()
    for i in range(2):
        ref.write(want[i], ks[i], slots, x[i], code)
    check_cache(cache, want, ks)
    return cache


def ragged_slots(rng, blocks, bt, runs):
    """Runs of rows at (cached length, new length), each sequence in blocks of its own."""
    order, slots, at = rng.permutation(blocks), [], 0
    for cached, new in runs:
        pages = order[at:at + -(-(cached + new) // bt)]
        at += len(pages)
        assert at <= blocks
        slots += [int(pages[p // bt]) * bt + p % bt for p in range(cached, cached + new)]
    return slots


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("heads,bt,dim,runs", [
    (1, 16, 64, [(0, 1)]), (4, 16, 64, [(5, 1), (16, 1), (31, 1), (0, 1)]),
    (2, 16, 128, [(0, 48), (3, 50), (15, 1), (7, 9)]), (3, 32, 64, [(0, 33), (31, 2), (1, 31)]),
    (2, 64, 128, [(10, 200), (0, 64)]), (1, 128, 64, [(100, 300)]), (2, 256, 128, [(0, 256), (255, 2)])])
def test_write(gpu, code, io, heads, bt, dim, runs):
    rng = np.random.default_rng(bt + dim + len(runs))
    slots = ragged_slots(rng, 24, bt, runs)
    x = rng.standard_normal((2, len(slots), heads, dim)) * np.exp(rng.standard_normal((2, len(slots), 1, 1)))
    run_write(gpu, code, 24, heads, bt, dim, slots, x, io)


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("bt", [16, 64])
def test_write_of_many_rows(gpu, code, bt):
    """Enough rows for teams that look through several, with padding and holes among them."""
    rng = np.random.default_rng(5)
    slots = np.array(ragged_slots(rng, 2400 * 16 // bt + 200, bt, [(0, 3000), (7, 1), (40, 2001)] + [(9, 1)] * 70))
    slots[rng.integers(0, len(slots), 40)] = -1
    slots = np.concatenate((slots, [-1] * 20))
    x = rng.standard_normal((2, len(slots), 2, 64))
    run_write(gpu, code, 2400 * 16 // bt + 200, 2, bt, 64, slots, x, "f32")


@pytest.mark.parametrize("code", [E4M3, INT8])
def test_write_of_border_values(gpu, code):
    """Ties, the format's largest and smallest values, subnormals, zeros, the type's extremes."""
    top = ref.TOP[code]
    tiny, huge = np.float32(2.0 ** -149), np.finfo(np.float32).max
    rows = np.zeros((13, 64), np.float32)
    rows[0, :9] = [top, -top, top / 2, 1.5, 2.5, 3.5, -0.5, 0.5, 1.0]
    rows[1, :5] = [2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -6, top]
    rows[2, :2] = [np.nextafter(np.float32(top), np.float32(huge)), 1.0]
    rows[4, 0] = tiny
    rows[5, :2] = [2.0 ** -126, -(2.0 ** -130)]
    rows[6, :2] = [huge, 1.0]
    rows[7, :3] = [17.0, 18.0, 19.0]
    rows[8] = np.linspace(-top, top, 64)
    rows[9] = 2.0 ** np.linspace(-20, 8, 64)
    rows[10, 0], rows[11, 0], rows[12, 0] = -huge, 448.0, 127.0
    slots = [16 * i for i in range(13)]
    x = np.stack([rows, -rows])[:, :, None, :]
    run_write(gpu, code, 16, 1, 16, 64, slots, x, "f32")
    run_write(gpu, code, 16, 1, 16, 64, [s + 3 for s in slots], x, "f32", seed=2)


def test_write_from_rows_of_a_wider_projection(gpu):
    rng = np.random.default_rng(8)
    slots = ragged_slots(rng, 8, 16, [(0, 20), (9, 5)])
    for io in ("f32", "bf16"):
        run_write(gpu, E4M3, 8, 2, 16, 64, slots, rng.standard_normal((2, len(slots), 2, 64)), io, stride=400)


@pytest.mark.parametrize("code", [E4M3, INT8])
def test_write_reports_what_is_not_finite(gpu, code):
    rng = np.random.default_rng(9)
    x = rng.standard_normal((2, 20, 2, 64))
    gpu.take_status()
    run_write(gpu, code, 4, 2, 16, 64, list(range(3, 23)), x, "f32")
    assert gpu.take_status()[0] == gpu.OK
    x[0, 4, 1, 7], x[0, 5, 0, 3], x[1, 19, 1, 63] = np.inf, np.nan, -np.inf
    x[1, 2] = np.nan
    run_write(gpu, code, 4, 2, 16, 64, list(range(3, 23)), x, "f32")
    rc, message = gpu.take_status()
    assert rc == gpu.ERR_RANGE and "8-bit" in message
    assert gpu.take_status()[0] == gpu.OK


@pytest.mark.parametrize("bt", [16, 64, 256])
def test_write_of_runs_that_windows_cut(gpu, bt):
    """Runs across the 64 rows that a wavefront sees at once, blocks that follow each other in the
    cache, several runs of one block with skipped rows between them, at every phase."""
    rng = np.random.default_rng(bt)
    for lead in (0, 1, 37, 63, 64, 65):
        slots = [-1] * lead + list(range(5, 5 + 3 * bt)) + [-1] * 62 + [3 * bt + 9, 3 * bt + 10]
        slots += [6 * bt, 6 * bt + 1, -1, -1, 6 * bt + 7, 6 * bt + 3, 6 * bt + 4, 2 ** 40, 8 * bt + bt - 1]
        x = rng.standard_normal((2, len(slots), 1, 64)) * np.exp(rng.standard_normal((2, len(slots), 1, 1)))
        run_write(gpu, E4M3 if lead % 2 else INT8, 10, 1, bt, 64, slots, x, "f32", seed=lead)
    slots = [s for b in rng.permutation(300) for s in range(b * bt, b * bt + bt)] if bt == 16 else list(range(9 * bt))
    x = rng.standard_normal((2, len(slots), 4, 64))
    run_write(gpu, E4M3, 300 if bt == 16 else 9, 4, bt, 64, slots, x, "bf16")


@pytest.mark.parametrize("bt", [16, 128])
@pytest.mark.parametrize("code", [E4M3, INT8])
def test_write_of_a_slot_twice(gpu, code, bt):
    """Each is a run of its own; a later one finds the tokens in front of it as the earlier left them."""
    rng = np.random.default_rng(88)
    slots = np.array([5, 6, 6, 7, 7, 7, bt + 3, bt, bt, bt + 1], np.int64)
    x = [rng.standard_normal((len(slots), 2, 64)) * np.exp2(rng.integers(-6, 7, (len(slots), 1, 1))) for _ in range(2)]
    run_write(gpu, code, 4, 2, bt, 64, slots, x, "f32")


def test_write_skips_slots_outside_the_cache(gpu):
    rng = np.random.default_rng(10)
    slots = [-1, 5, 6, 64, 2 ** 40, -2 ** 40, 63, 7, 8]
    run_write(gpu, E4M3, 4, 2, 16, 64, slots[:7], rng.standard_normal((2, 7, 2, 64)), "f32")


# ------------------------------------------------------------- decode

def laid_out(rng, code, lens, heads, bt, dim, levels=(-9, -4), spare=2):
    """A cache with sequences of these lengths; whatever is not a live token is poisoned: NaN
    codes (-128 for integers) and NaN scales.  Returns codes, scales, tables."""
    need = [-(-max(n, 0) // bt) for n in lens]
    blocks = sum(need) + spare
    codes, scales = random_cache(rng, code, blocks, heads, bt, dim)
    scales = (2.0 ** rng.uniform(*levels, scales.shape)).astype(np.float32)
    order = rng.permutation(blocks)
    tables = np.full((len(lens), max(max(need), 1) + 1), 2 ** 30, np.int32)
    live = np.zeros((blocks, bt), bool)
    at = 0
    for b, n in enumerate(lens):
        tables[b, :need[b]] = order[at:at + need[b]]
        for i, blk in enumerate(order[at:at + need[b]]):
            live[blk, :max(min(n - i * bt, bt), 0)] = True
        at += need[b]
    codes[:, :, :, :, :] = np.where(live[None, :, None, :, None], codes, 0x7f if code == E4M3 else 0x80)
    scales[:, ~live.any(1)] = np.nan
    return codes, scales, tables


def values_of(codes, scales, code, table, n, bt):
    """K, V [n][heads][dim] of one sequence in 64 bits."""
    lut, out = ref.code_values(code), []
    for i in range(2):
        pages = [lut[codes[i, b]] * scales[i, b].astype(np.float64)[:, None, None] for b in table[:-(-n // bt)]]
        out.append(np.concatenate(pages, 1)[:, :n].transpose(1, 0, 2) if pages else np.zeros((0,) + codes.shape[2:3] + codes.shape[4:]))
    return out


def unit_of(scales, code):
    """The largest magnitude that V's scales allow."""
    return float(np.nanmax(scales[1])) * ref.TOP[code]


def check_decode(gpu, code, lens, q_heads, heads, bt, dim, io="f32", seed=0, q_scale=1.0, max_ctx=None,
                 levels=(-9, -4), scale=0.0, softcap=0.0, window=0, slopes=None, drop=(), q=None, workspace=None):
    rng = np.random.default_rng(seed)
    codes, scales, tables = laid_out(rng, code, lens, heads, bt, dim, levels)
    presents = []
    for b, n in enumerate(lens):
        present = np.ones(max(n, 0), bool)
        for page, bad in drop:
            if page * bt < n:
                present[page * bt:(page + 1) * bt] = False
        presents.append(present)
    whole = tables.copy()
    for page, bad in drop:
        if page < tables.shape[1]:
            tables[:, page] = bad
    if q is None:
        q = rng.standard_normal((len(lens), q_heads, dim)) * q_scale
    q = bf16(q) if io == "bf16" else q.astype(np.float32).astype(np.float64)
    dtype = torch.bfloat16 if io == "bf16" else torch.float32
    cache = gpu_cache(gpu, codes, scales, code)
    dq = dev(q, dtype)
    out = torch.full_like(dq, float("nan"))
    options = gpu.ScoreOptions(scale, softcap, window, None if slopes is None else dev(slopes, torch.float32))
    ws = gpu.kv8_decode(cache, dq, dev(tables), dev(np.asarray(lens, np.int32)), out, max_ctx=max_ctx,
                        options=options, workspace=workspace)
    got = out.double().cpu().numpy()
    if ws is not None:  # the counters, at the front, are back at zero
        assert not ws[:16384].any()
    slopes64 = None if slopes is None else np.asarray(slopes, np.float32).astype(np.float64)
    for b, n in enumerate(lens):
        if n <= 0:
            assert not got[b].any()
            continue
        k, v = values_of(codes, scales, code, whole[b], n, bt)
        want, bound = ref.attention(q[b:b + 1], k, v, [n - 1], scale, softcap, window, slopes64, present=presents[b],
                                    unit=unit_of(scales, code))
        if io == "bf16":
            bound = bound + np.abs(want) * BF16_HALF_STEP + 2.0 ** -133
        err = np.abs(got[b] - want[0])
        assert (err <= bound[0]).all(), (b, n, float((err / bound[0]).max()), float(err.max()))
    return got


SHAPES = [(32, 4, 64), (32, 8, 128), (12, 12, 64), (8, 2, 128), (5, 1, 64), (40, 2, 64), (34, 2, 128)]


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("q_heads,heads,dim", SHAPES)
@pytest.mark.parametrize("lens,bt", [([1], 16), ([2, 1, 15, 16, 17], 16), ([63, 64, 65, 129], 32),
                                     ([700], 64), ([300, 1, 1030, 257], 256)])
def test_decode(gpu, code, q_heads, heads, dim, lens, bt):
    check_decode(gpu, code, lens, q_heads, heads, bt, dim)


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("q_heads,heads,dim", [(32, 4, 64), (32, 8, 128)])
def test_decode_bf16(gpu, code, q_heads, heads, dim):
    check_decode(gpu, code, [500, 77, 1], q_heads, heads, 16, dim, io="bf16")


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch", [30, 130])
def test_decode_of_batches(gpu, dim, batch):
    """The form that lays all segments end to end: ragged lengths, padded entries, one long one."""
    rng = np.random.default_rng(batch)
    lens = rng.integers(1, 700, batch)
    lens[3], lens[7], lens[11], lens[12], lens[-1] = 0, 5000, 1, -3, 0
    check_decode(gpu, E4M3, lens.tolist(), 8, 4, 16, dim, seed=3)


def test_decode_of_more_sequences_than_a_launch_takes(gpu):
    rng = np.random.default_rng(1)
    check_decode(gpu, INT8, rng.integers(0, 40, 1100).tolist(), 4, 2, 16, 64)


@pytest.mark.parametrize("lens,heads", [([9000], 2), ([20000, 3], 1)])
def test_decode_of_long_contexts(gpu, lens, heads):
    check_decode(gpu, E4M3, lens, 8 * heads, heads, 16, 64)
    check_decode(gpu, INT8, lens, 4 * heads, heads, 64, 128)


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("options", [
    dict(softcap=30.0), dict(softcap=2.0, q_scale=6.0), dict(softcap=0.5, q_scale=30.0), dict(slopes=True),
    dict(slopes=True, softcap=20.0), dict(window=1), dict(window=64), dict(window=100, slopes=True),
    dict(scale=0.37), dict(scale=3.0, softcap=50.0)])
def test_decode_options(gpu, code, options):
    o = dict(options)
    if o.get("slopes"):
        o["slopes"] = 2.0 ** (-8.0 * np.arange(1, 9) / 8)
    check_decode(gpu, code, [1, 64, 400, 99, 1000], 8, 2, 16, 64, **o)
    check_decode(gpu, code, [130] * 40, 8, 2, 32, 128, **o)


def test_decode_does_not_depend_on_max_ctx(gpu):
    """max_ctx shapes the launch: bounds above and below the lengths give the same attention."""
    for max_ctx in (1, 100, 4000, 100000):
        check_decode(gpu, E4M3, [900, 33], 8, 2, 16, 64, max_ctx=max_ctx)
        check_decode(gpu, E4M3, [900, 33] * 40, 8, 2, 16, 64, max_ctx=max_ctx)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("code,options", [(E4M3, {}), (INT8, {}), (E4M3, dict(softcap=30.0)), (INT8, dict(softcap=30.0))])
def test_decode_of_batches_that_may_be_large(gpu, code, options, dim):
    """Bounds from which a launch reads past the memory-side cache."""
    lens = np.random.default_rng(23).integers(0, 700, 40).tolist()
    check_decode(gpu, code, lens, 8, 2, 32, dim, max_ctx=1 << 20, **options)


def test_decode_skips_pages_that_are_no_blocks(gpu):
    """Entries past the cache or negative, at a tile's edge and inside it, in the middle and at the end."""
    for drop in ([(1, -1)], [(0, 2 ** 31 - 1), (5, -7)], [(4, 10 ** 6), (5, -1), (6, -1), (7, -1)],
                 [(i, -1) for i in range(100)]):
        check_decode(gpu, E4M3, [160, 97, 16], 8, 2, 16, 64, drop=drop)


def test_decode_of_scales_far_apart(gpu):
    """V scales from 2^-60 to 2^40 and K scales that make one block's scores decide."""
    check_decode(gpu, E4M3, [300, 40], 8, 2, 16, 64, levels=(-9, 0), q_scale=0.5)
    check_decode(gpu, INT8, [300, 40], 8, 2, 16, 64, levels=(-60, -50))
    check_decode(gpu, INT8, [300, 40], 8, 2, 16, 64, levels=(30, 40), q_scale=1e-11)


def test_decode_of_extreme_q(gpu):
    """q is carried relative to its largest value: magnitudes beyond binary16 are no special case."""
    rng = np.random.default_rng(4)
    q = rng.standard_normal((2, 8, 64)) * np.exp(3 * rng.standard_normal((2, 8, 64)))
    check_decode(gpu, E4M3, [200, 40], 8, 2, 16, 64, q=q * 1e6, scale=1e-7)
    check_decode(gpu, E4M3, [200, 40], 8, 2, 16, 64, q=q * 1e-30, scale=1e29)
    check_decode(gpu, E4M3, [200, 40], 8, 2, 16, 64, q=q * 0)


def test_decode_keeps_nan_to_its_head(gpu):
    rng = np.random.default_rng(6)
    codes, scales, tables = laid_out(rng, E4M3, [300, 70], 2, 16, 64)
    cache = gpu_cache(gpu, codes, scales, E4M3)
    q = torch.randn(2, 8, 64, device="cuda")
    clean, out = torch.empty_like(q), torch.empty_like(q)
    lens, tables = dev(np.array([300, 70], np.int32)), dev(tables)
    gpu.kv8_decode(cache, q, tables, lens, clean)
    q[0, 3, 5], q[1, 6, 1] = float("nan"), float("inf")
    gpu.kv8_decode(cache, q, tables, lens, out)
    assert out[0, 3].isnan().all() and out[1, 6].isnan().all()
    out[0, 3], out[1, 6] = clean[0, 3], clean[1, 6]
    assert torch.equal(out, clean)


def test_decode_of_rows_of_a_wider_projection(gpu):
    rng = np.random.default_rng(12)
    codes, scales, tables = laid_out(rng, E4M3, [100, 30], 2, 16, 64)
    cache = gpu_cache(gpu, codes, scales, E4M3)
    wide = torch.randn(2, 8 * 64 + 256, device="cuda")
    q = wide[:, :8 * 64].view(2, 8, 64)
    lens, tables = dev(np.array([100, 30], np.int32)), dev(tables)
    a, b = torch.empty(2, 8, 64, device="cuda"), torch.empty(2, 8, 64, device="cuda")
    gpu.kv8_decode(cache, q, tables, lens, a)
    gpu.kv8_decode(cache, q.contiguous(), tables, lens, b)
    assert torch.equal(a, b)


def test_decode_behind_four_gib(gpu):
    """Blocks whose offsets pass 32 bits are read and written where they are."""
    blocks, heads, bt, dim = 4_400_000_000 // (4 * 256 * 128), 4, 256, 128
    cache = gpu.Kv8Cache.empty(blocks, heads, bt, dim)
    rng = np.random.default_rng(2)
    table = np.array([blocks - 1, 3, blocks - 2], np.int32)
    n = 600
    slots = np.array([int(table[p // bt]) * bt + p % bt for p in range(n)])
    x = rng.standard_normal((2, n, heads, dim)).astype(np.float32)
    gpu.kv8_write(cache, dev(slots), dev(x[0]), dev(x[1]))
    codes = np.zeros((2, 3, heads, bt, dim), np.uint8)
    scales = np.zeros((2, 3, heads))
    local = np.arange(n)
    for i in range(2):
        ref.write(codes[i], scales[i], local, x[i], E4M3)
    for i, t in enumerate((cache.k, cache.v)):
        got = t[torch.from_numpy(table).long().cuda()].cpu().numpy()
        live = got.transpose(0, 2, 1, 3).reshape(-1, heads, dim)[:n]
        want = codes[i].transpose(0, 2, 1, 3).reshape(-1, heads, dim)[:n]
        assert np.array_equal(np.where((live & 127) == 0, 0, live), np.where((want & 127) == 0, 0, want))
    q = rng.standard_normal((1, 8, dim)).astype(np.float32)
    out = torch.empty(1, 8, dim, device="cuda")
    gpu.kv8_decode(cache, dev(q), dev(table[None]), dev(np.array([n], np.int32)), out)
    k, v = values_of(codes, scales, E4M3, np.arange(3), n, bt)
    want, bound = ref.attention(q.astype(np.float64), k, v, [n - 1], unit=unit_of(scales, E4M3))
    assert (np.abs(out.cpu().numpy() - want) <= bound).all()


def test_decode_in_graphs_and_streams(gpu):
    """Two captured calls with workspaces of their own, replayed with new lengths between eager work."""
    rng = np.random.default_rng(7)
    lens = [3000, 500, 1, 900]
    codes, scales, tables = laid_out(rng, E4M3, lens, 2, 16, 64)
    cache = gpu_cache(gpu, codes, scales, E4M3)
    q = torch.randn(4, 8, 64, device="cuda")
    tables, dlens = dev(tables), dev(np.asarray(lens, np.int32))
    outs = [torch.empty_like(q) for _ in range(2)]
    ws = [gpu.alloc_workspace(gpu.kv8_decode_workspace_size(cache, 4, 8, 3000)) for _ in range(2)]
    graphs, side = [], torch.cuda.Stream()
    for o, w in zip(outs, ws):
        g = torch.cuda.CUDAGraph()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(g, stream=side):
            gpu.kv8_decode(cache, q, tables, dlens, o, max_ctx=3000, workspace=w)
        graphs.append(g)
    torch.cuda.synchronize()
    for step in range(4):
        dlens.copy_(torch.tensor([3000 - 700 * step, 500, 1 + step, 900 - step], dtype=torch.int32))
        q.copy_(torch.randn(4, 8, 64))
        eager = torch.empty_like(q)
        gpu.kv8_decode(cache, q, tables, dlens, eager, max_ctx=3000)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        # as bits: where a length grows into rows that were never written, NaN is the answer
        assert torch.equal(outs[0].view(torch.int32), eager.view(torch.int32)), step
        assert torch.equal(outs[1].view(torch.int32), eager.view(torch.int32)), step
        assert eager[0].isfinite().all() and eager[3].isfinite().all()
        for o in outs:
            o.zero_()


def test_decode_gives_the_same_bits_every_time(gpu):
    rng = np.random.default_rng(13)
    lens = rng.integers(1, 4000, 48)
    codes, scales, tables = laid_out(rng, E4M3, lens.tolist(), 4, 16, 64)
    cache, q = gpu_cache(gpu, codes, scales, E4M3), torch.randn(48, 32, 64, device="cuda")
    tables, dlens = dev(tables), dev(lens.astype(np.int32))
    first = torch.empty_like(q)
    ws = gpu.kv8_decode(cache, q, tables, dlens, first, max_ctx=4000)
    for _ in range(20):
        out = torch.full_like(q, float("nan"))
        gpu.kv8_decode(cache, q, tables, dlens, out, max_ctx=4000, workspace=ws)
        assert torch.equal(out, first)


# ------------------------------------------------------------- together

@pytest.mark.parametrize("code,io", [(E4M3, "f32"), (INT8, "bf16")])
def test_serving_steps(gpu, code, io):
    """Prompts admitted into an empty cache, then decode steps whose tokens are appended to it, with
    the map's slots all the way; a sequence ends, and a new one takes its place and blocks."""
    rng = np.random.default_rng(21)
    heads, q_heads, bt, dim, batch, pages = 2, 8, 16, 64, 5, 12
    dtype = torch.float32 if io == "f32" else torch.bfloat16
    cache = gpu.Kv8Cache.empty(80, heads, bt, dim, code)
    free = list(rng.permutation(80))
    tables = np.full((batch, pages), -1, np.int32)
    codes = np.zeros((2, 80, heads, bt, dim), np.uint8)
    scales = np.zeros((2, 80, heads))
    lens = np.zeros(batch, np.int32)
    for step in range(8):
        new = np.ones(batch, np.int32) if step else np.array([30, 1, 16, 47, 100], np.int32)
        if step == 4:  # sequence 2 ends, another prompt takes its row
            free += [b for b in tables[2] if b >= 0]
            tables[2], lens[2], new[2] = -1, 0, 33
        n_rows = int(new.sum()) + 3
        got_t, m = run_map(gpu, lens, new, free, tables, bt, 80, n_rows)
        want = ref.batch_map(lens, new, free, tables, bt, 80, n_rows)
        assert np.array_equal(got_t, tables) and np.array_equal(m["slots"], want[2])
        free = free[int(m["counts"][0]):]
        lens = m["ctx_lens"]
        x = rng.standard_normal((2, n_rows, heads, dim)) * (1 + 0.2 * step)
        x = bf16(x) if io == "bf16" else x.astype(np.float32).astype(np.float64)
        gpu.kv8_write(cache, dev(m["slots"]), dev(x[0], dtype), dev(x[1], dtype))
        for i in range(2):
            ref.write(codes[i], scales[i], m["slots"], x[i], code)
        check_cache(cache, codes, scales)
        q = rng.standard_normal((batch, q_heads, dim))
        q = bf16(q) if io == "bf16" else q.astype(np.float32).astype(np.float64)
        out = torch.empty(batch, q_heads, dim, dtype=dtype, device="cuda")
        gpu.kv8_decode(cache, dev(q, dtype), dev(tables), dev(lens), out)
        for b in range(batch):
            k, v = values_of(codes, scales, code, tables[b], int(lens[b]), bt)
            want, bound = ref.attention(q[b:b + 1], k, v, [lens[b] - 1], unit=unit_of(scales, code))
            bound = bound + (np.abs(want) * BF16_HALF_STEP if io == "bf16" else 0)
            assert (np.abs(out[b].double().cpu().numpy() - want[0]) <= bound[0]).all()


# ------------------------------------------------------------- refusals

def refused(gpu, code, call):
    with pytest.raises(gpu.NyionError) as e:
        call()
    assert e.value.code == code, e.value


def test_refusals(gpu):
    cache = gpu.Kv8Cache.empty(8, 2, 16, 64)
    q = torch.zeros(2, 8, 64, device="cuda")
    out, tables = torch.empty_like(q), torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    lens = torch.full((2,), 2000, dtype=torch.int32, device="cuda")
    big = torch.zeros(2, 400, dtype=torch.int32, device="cuda")
    INV, UNS, WS = gpu.ERR_INVALID, gpu.ERR_UNSUPPORTED, gpu.ERR_WORKSPACE
    dec = lambda **k: gpu.kv8_decode(**{**dict(cache=cache, q=q, block_tables=tables, ctx_lens=lens, out=out,  # noqa: E731
                                               max_ctx=2000), **k})
    small = torch.zeros(256, dtype=torch.uint8, device="cuda")
    refused(gpu, WS, lambda: dec(block_tables=big, workspace=small))
    ws = gpu.alloc_workspace(1 << 22)
    refused(gpu, INV, lambda: dec(workspace=ws[8:]))
    refused(gpu, INV, lambda: dec(q=q[:, :7]))
    refused(gpu, INV, lambda: dec(q=q[:1]))
    refused(gpu, INV, lambda: dec(q=q.half()))
    refused(gpu, INV, lambda: dec(out=out.bfloat16()))
    refused(gpu, INV, lambda: dec(ctx_lens=lens.long()))
    refused(gpu, INV, lambda: dec(ctx_lens=lens.cpu()))
    refused(gpu, INV, lambda: dec(max_ctx=0))
    refused(gpu, INV, lambda: dec(options=gpu.ScoreOptions(softcap=-1.0)))
    refused(gpu, INV, lambda: dec(options=gpu.ScoreOptions(scale=float("nan"))))
    refused(gpu, INV, lambda: dec(options=gpu.ScoreOptions(softcap=1e-42)))
    refused(gpu, INV, lambda: dec(options=gpu.ScoreOptions(scale=3e38)))
    refused(gpu, INV, lambda: dec(options=gpu.ScoreOptions(prefix_lens=lens)))
    refused(gpu, INV, lambda: dec(options=gpu.ScoreOptions(slopes=torch.zeros(7, device="cuda"))))
    wide = torch.zeros(2, 8 * 64 + 2, device="cuda")
    refused(gpu, INV, lambda: dec(q=wide[:, 1:513].view(2, 8, 64)))
    refused(gpu, UNS, lambda: gpu.kv8_write(gpu.Kv8Cache.empty(8, 2, 8, 64), torch.zeros(1, dtype=torch.int64, device="cuda"),
                                            torch.zeros(1, 2, 64, device="cuda"), torch.zeros(1, 2, 64, device="cuda")))
    refused(gpu, UNS, lambda: gpu.kv8_write(gpu.Kv8Cache.empty(8, 2, 16, 96), torch.zeros(1, dtype=torch.int64, device="cuda"),
                                            torch.zeros(1, 2, 96, device="cuda"), torch.zeros(1, 2, 96, device="cuda")))
    k = torch.zeros(3, 2, 64, device="cuda")
    refused(gpu, INV, lambda: gpu.kv8_write(cache, torch.zeros(2, dtype=torch.int64, device="cuda"), k, k))
    refused(gpu, INV, lambda: gpu.kv8_write(cache, torch.zeros(3, dtype=torch.int32, device="cuda"), k, k))
    refused(gpu, INV, lambda: gpu.kv8_write(cache, torch.zeros(3, dtype=torch.int64, device="cuda"), k, k.bfloat16()))
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    one = i32(1)
    refused(gpu, INV, lambda: gpu.batch_map(one, i32(1), i32(4), i32(1, 4), 12, 8, i32(1), i32(2),
                                            torch.zeros(3, dtype=torch.int64, device="cuda"), i32(3), i32(2)))
    refused(gpu, INV, lambda: gpu.batch_map(one, i32(1), i32(4), i32(1, 4), 16, 8, one, i32(2),
                                            torch.zeros(3, dtype=torch.int64, device="cuda"), i32(3), i32(2)))
    refused(gpu, UNS, lambda: gpu.batch_map(i32(4097), i32(4097), i32(4), i32(4097, 1), 16, 8, i32(4097), i32(4098),
                                            torch.zeros(3, dtype=torch.int64, device="cuda"), i32(3), i32(2)))


def test_nothing_to_write_is_no_error(gpu):
    cache = gpu.Kv8Cache.empty(2, 2, 16, 64)
    none = torch.zeros(0, 2, 64, device="cuda")
    gpu.kv8_write(cache, torch.zeros(0, dtype=torch.int64, device="cuda"), none, none)
    torch.cuda.synchronize()
