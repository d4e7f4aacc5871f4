"""GPU: the quantised attention over packed prompts and over a paged cache, the cache write and the paging plan against their definitions in 64-bit integers.
Everything is integers: results are equal, or wrong."""
import ctypes as C

import numpy as np
import pytest

from _attention_ref import ONE, attend, mask_weighs, plan, prompt
from _dev import Dev, hip, ok, workspace

pytestmark = pytest.mark.gpu
MARK = 123456789


def values(rng, shape, sigma=1.0):
    """activations at scale 2^14, one channel in eight four times as large"""
    x = rng.normal(0, sigma, shape)
    x[..., ::8] *= 4
    return np.clip(np.round(x * ONE), -(1 << 18), (1 << 18) - 1).astype(np.int32)


def any_int32(rng, shape):
    x = rng.integers(-(1 << 31), 1 << 31, size=shape, dtype=np.int64)
    return np.where(rng.random(shape) < 0.1, rng.choice([-(1 << 31), (1 << 31) - 1, 0, -1, 1 << 23, -(1 << 23)], size=shape), x).astype(np.int32)


# Which kernels take a call goes by what the host knows of it: the rows of the arrays (prompts) and the columns of the table (cached).  Rows behind the last
# sequence, and columns that no sequence uses, send the same sequences through each: all scores in LDS; tiles; tiles with more keys than their e is held for;
# keys split over workgroups.
PROMPT_ROWS = (0, 2100, 16500)
CACHED_KEYS = (0, 1100, 4200, 16600)


def run_prompt(A, q, k, v, lens, mul=ONE, causal=True, pads=PROMPT_ROWS):
    import jolt_atlas_amd.attention as T
    n, H, d = q.shape
    at = T.Attention(H, k.shape[1], d, mul, causal)
    cu = Dev(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))
    got = None
    for rows in pads:
        rows = max(rows, n)
        more = lambda x, fill: np.concatenate([x, np.full((rows - n,) + x.shape[1:], fill, np.int32)])  # noqa: E731
        out = Dev(np.full((rows, H, d), MARK, np.int32))
        ws = workspace(at.prompt_workspace_bytes(len(lens), rows))
        assert at.prompt(Dev(more(q, -(1 << 31))), Dev(more(k, -(1 << 31))), Dev(more(v, -(1 << 31))), cu, out, ws) is out
        x = out.numpy()
        assert (x[n:] == MARK).all(), rows
        assert got is None or np.array_equal(got, x[:n]), rows
        got = x[:n]
    return got


SHAPES = [(1, 1, 1), (4, 4, 4), (4, 4, 16), (4, 2, 20), (6, 2, 32), (5, 5, 33), (16, 16, 64), (8, 2, 64), (3, 1, 80), (8, 1, 96), (12, 4, 128), (7, 7, 100), (2, 1, 192), (3, 3, 256), (5, 1, 255)]


@pytest.mark.parametrize("H,KV,d", SHAPES)
def test_prompt(atlas, H, KV, d):
    rng = np.random.default_rng(H * 1000 + d)
    lens = [37, 0, 1, 64, 130, 5, 0, 33, 32, 31, 0]
    n = sum(lens)
    q, k, v = values(rng, (n, H, d)), values(rng, (n, KV, d)), values(rng, (n, KV, d))
    mul = int(round(ONE / np.sqrt(d)))
    got = run_prompt(atlas, q, k, v, lens, mul)
    assert np.array_equal(got, prompt(q, k, v, lens, mul))


@pytest.mark.parametrize("H,KV,d,n", [(2, 1, 64, 700), (2, 2, 128, 513), (1, 1, 16, 1025), (4, 1, 80, 300), (1, 1, 256, 290)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("mul", [ONE, 1448, 1])
def test_prompt_longer(atlas, H, KV, d, n, causal, mul):
    rng = np.random.default_rng(n)
    lens = [n, 77]
    N = sum(lens)
    q, k, v = values(rng, (N, H, d), 0.4 if mul == ONE else 1.0), values(rng, (N, KV, d)), values(rng, (N, KV, d))
    assert np.array_equal(run_prompt(atlas, q, k, v, lens, mul, causal), prompt(q, k, v, lens, mul, causal))


@pytest.mark.parametrize("lens", [[1], [0], [0, 0, 0], [1, 1, 1, 1], [2, 3], [63], [64], [65], [127, 1], [128], [129], [1] * 300, [0] * 70 + [3] + [0] * 70])
def test_prompt_lengths(atlas, lens):
    rng = np.random.default_rng(len(lens))
    n = sum(lens) + 3                       # rows behind the last sequence: neither read nor written
    q, k, v = values(rng, (n, 4, 16)), values(rng, (n, 2, 16)), values(rng, (n, 2, 16))
    got = run_prompt(atlas, q, k, v, lens, 4096)
    assert np.array_equal(got[:n - 3], prompt(q[:n - 3], k[:n - 3], v[:n - 3], lens, 4096))
    assert (got[n - 3:] == MARK).all()


def test_prompt_without_rows_or_sequences(atlas):
    import jolt_atlas_amd.attention as T
    at = T.Attention(2, 1, 8)
    e = lambda h: Dev(np.zeros((0, h, 8), np.int32))  # noqa: E731
    at.prompt(e(2), e(1), e(1), Dev(np.zeros(4, np.int32)), e(2), workspace(at.prompt_workspace_bytes(3, 0)))
    x = np.full((5, 2, 8), MARK, np.int32)
    out = Dev(x)
    at.prompt(Dev(x.copy()), Dev(x[:, :1]), Dev(x[:, :1]), Dev(np.zeros(1, np.int32)), out, workspace(at.prompt_workspace_bytes(0, 5)))
    assert (out.numpy() == MARK).all()


@pytest.mark.parametrize("H,KV,d,n", [(2, 1, 16, 70), (2, 2, 64, 40), (1, 1, 128, 130), (3, 1, 37, 33)])
@pytest.mark.parametrize("kind", ["any", "edge", "wide_q", "wide_k", "wide_v", "large"])
def test_prompt_of_any_int32(atlas, H, KV, d, n, kind):
    """operands beyond what three signed bytes hold, sums that wrap, scores that clamp"""
    rng = np.random.default_rng(d + n)
    q, k, v = values(rng, (n, H, d)), values(rng, (n, KV, d)), values(rng, (n, KV, d))
    if kind == "any":
        q, k, v = any_int32(rng, q.shape), any_int32(rng, k.shape), any_int32(rng, v.shape)
    elif kind == "edge":                     # the borders of three signed bytes
        pick = lambda s: rng.choice([8355711, 8355712, -8421504, -8421505, 32639, 32640, -32896, 127, 128, -128, -129, 0], size=s).astype(np.int32)  # noqa: E731
        q, k, v = pick(q.shape), pick(k.shape), pick(v.shape)
    elif kind == "wide_q":
        q[n // 2, 0, d // 2] = (1 << 31) - 1
    elif kind == "wide_k":
        k[3, -1, 0] = -(1 << 31)
    elif kind == "wide_v":
        v[n - 1, 0, d - 1] = (1 << 31) - 1
    else:
        q, k, v = q * 20, k * 20, v * 20
    for mul in (ONE, 1448):
        assert np.array_equal(run_prompt(atlas, q, k, v, [n], mul), prompt(q, k, v, [n], mul))


# |q| |k| d = 2^45: the score is 2^31, one more than 32 bits hold, and the definition clamps it
BORDER = [(1, 23, 22), (16, 21, 20), (32, 20, 20), (64, 22, 17), (64, 23, 16), (64, 19, 20), (128, 23, 15), (256, 20, 17)]


@pytest.mark.parametrize("d,a,b", BORDER)
def test_prompt_scores_of_2_to_31(atlas, d, a, b):
    rng = np.random.default_rng(d)
    n = 70
    q, k, v = np.full((n, 2, d), -(1 << a), np.int32), np.zeros((n, 1, d), np.int32), values(rng, (n, 1, d))
    k[5], k[40] = -(1 << b), (1 << b) - 1                # one key at the border, one as far below
    assert int(q[0, 0].astype(np.int64) @ k[5, 0]) == 1 << 45
    for mul in (ONE, 1448):
        assert np.array_equal(run_prompt(atlas, q, k, v, [n], mul), prompt(q, k, v, [n], mul))


@pytest.mark.parametrize("d,a,b", BORDER)
@pytest.mark.parametrize("new", [1, 70])
def test_cached_scores_of_2_to_31(atlas, d, a, b, new):
    rng = np.random.default_rng(d)
    ck, cv, table, flat = paged(rng, [100], 1, d, 16, 32)
    ck[:] = 0
    ck[table[0, 0], 0, 3], ck[table[0, 1], 0, 2] = -(1 << b), (1 << b) - 1
    q = np.full((new, 2, d), -(1 << a), np.int32)
    assert np.array_equal(run_cached(q, ck, cv, table, [100], [new], 2048), want_cached(q, ck, cv, table, flat, [100], [new], 2048))


def test_prompt_scores_that_are_equal_or_far_apart(atlas):
    rng = np.random.default_rng(9)
    n, d = 257, 64
    q, k, v = values(rng, (n, 1, d)), np.zeros((n, 1, d), np.int32), values(rng, (n, 1, d))
    assert np.array_equal(run_prompt(atlas, q, k, v, [n]), prompt(q, k, v, [n]))            # all weights alike
    k[:] = values(rng, k.shape, 3.0)
    assert np.array_equal(run_prompt(atlas, q, k, v, [n]), prompt(q, k, v, [n]))            # one key takes all
    k[200:] = k[17]
    assert np.array_equal(run_prompt(atlas, q, k, v, [n]), prompt(q, k, v, [n]))            # the maximum many times
    v[:] = (1 << 22)
    assert np.array_equal(run_prompt(atlas, q, k, v, [n], 512), prompt(q, k, v, [n], 512))


@pytest.mark.parametrize("d,off", [(16, 0), (64, 1), (80, 3), (33, 2), (128, 1)])
def test_prompt_strides(atlas, d, off):
    """q, k, v as slices of one projection's output, at offsets that no vector load likes; out inside a larger array"""
    import jolt_atlas_amd.attention as T
    rng = np.random.default_rng(d)
    H, KV, lens = 4, 2, [45, 0, 70]
    n, width = sum(lens), (H + 2 * KV) * d + 7
    row = values(rng, (n, width))
    R = Dev(row)
    view = lambda at, h: R.view(at, (n, h, d), (width, d, 1))  # noqa: E731
    part = lambda at, h: row[:, at:at + h * d].reshape(n, h, d)  # noqa: E731
    at = T.Attention(H, KV, d, 2048)
    outer = Dev(np.full((H, n + 2, d + 5), MARK, np.int32))                                # heads outside of tokens
    out = outer.view((d + 5) + off, (n, H, d), (d + 5, (n + 2) * (d + 5), 1))
    at.prompt(view(off, H), view(off + H * d, KV), view(off + (H + KV) * d, KV), Dev(np.cumsum([0] + lens).astype(np.int32)), out, workspace(at.prompt_workspace_bytes(3, n)))
    want = prompt(part(off, H), part(off + H * d, KV), part(off + (H + KV) * d, KV), lens, 2048)
    full = np.full((H, n + 2, d + 5), MARK, np.int32)
    full[:, 1:n + 1, off:off + d] = want.transpose(1, 0, 2)
    assert np.array_equal(outer.numpy(), full)


# ------------------------------------------------------------------------------------------------------------- paged cache
def paged(rng, keys, KV, d, block, bits, spare=3, cols=None, sigma=None):
    """caches with random blocks for sequences of `keys`, their table, and the sequences' own keys and values"""
    up = [-(-k // block) for k in keys]
    n_blocks = sum(up) + spare
    dtype = np.int16 if bits == 16 else np.int32
    sigma = sigma or (0.4 if bits == 16 else 1.0)
    ck, cv = (np.clip(values(rng, (n_blocks, KV, block, d), sigma), -32768, 32767 if bits == 16 else 1 << 30).astype(dtype) for _ in range(2))
    ids = rng.permutation(n_blocks).astype(np.int32)
    table = np.full((len(keys), cols or max(up + [1])), -1, np.int32)
    at = 0
    for i, u in enumerate(up):
        table[i, :u] = ids[at:at + u]
        at += u
    flat = lambda c, i: c[table[i, :up[i]]].transpose(0, 2, 1, 3).reshape(-1, KV, d)[:keys[i]]  # noqa: E731
    return ck, cv, table, flat


def run_cached(q, ck, cv, table, keys, new, mul=ONE, causal=True, table_view=None, caps=CACHED_KEYS):
    import jolt_atlas_amd.attention as T
    n, H, d = q.shape
    at = T.Attention(H, ck.shape[1], d, mul, causal)
    cache = T.KVCache(Dev(ck), Dev(cv))
    cu, lens, dq = Dev(np.cumsum([0] + list(new)).astype(np.int32)), Dev(np.array(keys, np.int32)), Dev(q)
    got = None
    for cap in ((0,) if table_view else caps):
        tab = table_view
        if tab is None:
            cols = max(-(-cap // ck.shape[2]), table.shape[1])
            tab = Dev(np.concatenate([table, np.full((len(table), cols - table.shape[1]), 2 ** 31 - 1, np.int32)], axis=1))
        out = Dev(np.full(q.shape, MARK, np.int32))
        at.cached(dq, cu, lens, cache, tab, out, workspace(at.cached_workspace_bytes(len(new), n, cache, tab.shape[1])))
        x = out.numpy()
        assert got is None or np.array_equal(got, x), cap
        got = x
    return got


def want_cached(q, ck, cv, table, flat, keys, new, mul=ONE, causal=True):
    out, at = np.full(q.shape, MARK, np.int32), 0
    for i, (m, n) in enumerate(zip(keys, new)):
        lim = [max(0, min(m, m - n + j + 1)) if causal else m for j in range(n)]
        out[at:at + n] = attend(q[at:at + n], flat(ck, i), flat(cv, i), lim, mul)
        at += n
    return out


@pytest.mark.parametrize("H,KV,d", [(1, 1, 1), (4, 4, 16), (16, 16, 64), (8, 2, 128), (8, 1, 80), (32, 4, 64), (3, 1, 256), (5, 5, 33), (40, 1, 32)])
@pytest.mark.parametrize("bits", [32, 16])
@pytest.mark.parametrize("block", [1, 16, 64])
def test_cached_single_tokens(atlas, H, KV, d, bits, block):
    rng = np.random.default_rng(H * 100 + d + block)
    keys = [1, 2, 31, 32, 33, 100, 257, 64, 5]
    new = [1] * len(keys)
    ck, cv, table, flat = paged(rng, keys, KV, d, block, bits)
    q = values(rng, (len(keys), H, d))
    mul = int(round(ONE / np.sqrt(d)))
    assert np.array_equal(run_cached(q, ck, cv, table, keys, new, mul), want_cached(q, ck, cv, table, flat, keys, new, mul))


@pytest.mark.parametrize("H,KV,d,bits,block", [(4, 4, 16, 32, 16), (8, 2, 128, 32, 32), (8, 2, 64, 16, 8), (6, 2, 100, 32, 64), (2, 1, 256, 16, 128), (16, 2, 33, 32, 4), (8, 1, 128, 16, 16)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("many", [False, True])
def test_cached_chunks(atlas, H, KV, d, bits, block, causal, many):
    """several new tokens beside single ones, a request that pauses, a prompt without a past, more new tokens than keys (rows that see nothing)"""
    rng = np.random.default_rng(d)
    keys, new = ([90, 200, 33, 70, 300, 4, 0, 1], [17, 1, 33, 0, 70, 9, 2, 1]) if not many else ([300, 260, 7], [201, 120, 9])
    ck, cv, table, flat = paged(rng, keys, KV, d, block, bits)
    q = values(rng, (sum(new), H, d))
    mul = int(round(ONE / np.sqrt(d)))
    assert np.array_equal(run_cached(q, ck, cv, table, keys, new, mul, causal), want_cached(q, ck, cv, table, flat, keys, new, mul, causal))


@pytest.mark.parametrize("bits", [32, 16])
@pytest.mark.parametrize("new", [[1, 1], [3, 40]])
def test_cached_long(atlas, bits, new):
    rng = np.random.default_rng(11)
    keys = [9001, 4500]
    ck, cv, table, flat = paged(rng, keys, 2, 64, 32, bits)
    q = values(rng, (sum(new), 4, 64))
    assert np.array_equal(run_cached(q, ck, cv, table, keys, new, 2048), want_cached(q, ck, cv, table, flat, keys, new, 2048))


# The split path lays the units of 256 keys of all row tiles and kv heads behind each other, and each workgroup has the same share of that line
LINES = {
    "one_unit_more_than_workgroups": (2, 1, 32, [4864] * 27, [1] * 27),                        # 513 units for 512 workgroups
    "uneven_shares": (6, 2, 36, [3000, 517, 1, 0, 9000, 256, 257, 8200, 4095] * 5, [1, 2, 1, 1, 0, 1, 3, 1, 1] * 5),
    "several_units": (4, 4, 16, [5000 - 37 * i for i in range(45)], [1] * 45),
    "just_below_all_workgroups": (1, 1, 16, [16640] * 63, [1] * 63),                           # 4095 units for 512
    "all_workgroups": (16, 8, 32, [2049 + 7 * i for i in range(64)], [1 if i % 9 else 0 for i in range(64)]),
    "tiles_of_several_rows": (16, 2, 128, [4000, 900, 2500, 0, 3333] * 8, [5, 7, 0, 2, 9] * 8),
    "many_sequences": (4, 2, 32, [(i * 37) % 611 for i in range(1500)], [(1, 1, 0, 2, 1)[i % 5] for i in range(1500)]),
}


@pytest.mark.parametrize("bits", [32, 16])
@pytest.mark.parametrize("name", LINES)
def test_cached_shares_of_several_units(atlas, name, bits):
    import jolt_atlas_amd.attention as T
    H, KV, d, keys, new = LINES[name]
    rng = np.random.default_rng(len(keys) + bits)
    G = H // KV
    units = sum(-(-n * G // 16) * -(-k // 256) for k, n in zip(keys, new)) * KV
    tiles = sum(-(-n * G // 16) for n in new)
    assert {"one_unit_more_than_workgroups": units == 513, "uneven_shares": 512 < units < 4096 and units % 512, "several_units": 2048 < units < 4096, "just_below_all_workgroups": units == 4095,
            "all_workgroups": units > 4096 and units % 1024, "tiles_of_several_rows": 2048 < units < 4096, "many_sequences": tiles > 1024}[name]
    ck, cv, table, flat = paged(rng, keys, KV, d, 32, bits)
    n = sum(new)
    q, mul = values(rng, (n, H, d)), int(round(ONE / np.sqrt(d)))
    got = run_cached(q, ck, cv, table, keys, new, mul, caps=(4200,))
    at = np.cumsum([0] + new)
    some = range(len(keys)) if len(keys) < 70 else sorted({0, 1, 2, 3, len(keys) - 1, *rng.integers(0, len(keys), 250).tolist()})
    for i in some:
        if new[i]:
            limits = [max(0, keys[i] - new[i] + j + 1) for j in range(new[i])]
            assert np.array_equal(got[at[i]:at[i + 1]], attend(q[at[i]:at[i + 1]], flat(ck, i), flat(cv, i), limits, mul)), (i, keys[i], new[i])


def test_cached_pages_that_do_not_exist(atlas):
    """a table entry outside the cache holds no keys; keys behind the table's columns do not exist; lengths that make no sense give empty rows"""
    rng = np.random.default_rng(3)
    for new in ([1, 1, 1, 1], [2, 5, 40, 1]):
        keys = [100, 90, 80, 64]
        ck, cv, table, flat = paged(rng, keys, 2, 32, 16, 32)
        bad = table.copy()
        bad[0, 2], bad[1, 0], bad[2, :] = -7, ck.shape[0], 2 ** 31 - 1
        q = values(rng, (sum(new), 4, 32))
        want, at = np.zeros(q.shape, np.int32), 0
        for i, (m, n) in enumerate(zip(keys, new)):
            there = np.repeat((bad[i] >= 0) & (bad[i] < ck.shape[0]), 16)[:m]
            lim = [there & (np.arange(m) < m - n + j + 1) for j in range(n)]
            want[at:at + n] = attend(q[at:at + n], flat(ck, i), flat(cv, i), lim, 2896)
            at += n
        assert np.array_equal(run_cached(q, ck, cv, bad, keys, new, 2896), want)
        # the table cut to 3 columns: 48 keys are left of each sequence
        cut = Dev(table).view(0, (4, 3), (table.shape[1], 1))
        short = [48] * 4
        got = run_cached(q, ck, cv, None, keys, new, 2896, table_view=cut)
        assert np.array_equal(got, want_cached(q, ck, cv, table, lambda c, i: flat(c, i)[:48], short, new, 2896))
        assert (run_cached(q, ck, cv, table, [-5, 0, -(2 ** 31), 0], new, 2896) == 0).all()


@pytest.mark.parametrize("d", [32, 36, 64, 128, 256])
@pytest.mark.parametrize("new", [[1, 1, 1], [60, 90, 33]])
def test_cached_pages_that_do_not_exist_and_a_first_block_of_extremes(atlas, d, new):
    """whatever is read in the place of a page that is missing does not count: the cache's first block holds the largest operands, and no sequence has it"""
    rng = np.random.default_rng(d)
    keys = [150, 97, 33]
    ck, cv, table, flat = paged(rng, keys, 2, d, 16, 32)
    table = np.where(table >= 0, table + 1, -1).astype(np.int32)
    ends = np.array([-(1 << 31), (1 << 31) - 1], np.int32)
    first = lambda c: np.concatenate([rng.choice(ends, size=c[:1].shape).astype(np.int32), c])  # noqa: E731
    small = [ck, cv]
    ck, cv = first(ck), first(cv)
    table[0, 3], table[1, 0], table[2, 1] = -1, len(ck), -(1 << 31)
    q, want, at = values(rng, (sum(new), 8, d)), np.zeros((sum(new), 8, d), np.int32), 0
    for i, (m, n) in enumerate(zip(keys, new)):
        there = np.repeat((table[i] >= 0) & (table[i] < len(ck)), 16)[:m]
        lim = [there & (np.arange(m) < m - n + j + 1) for j in range(n)]
        want[at:at + n] = attend(q[at:at + n], flat(small[0], i), flat(small[1], i), lim, 1448)
        at += n
    assert np.array_equal(run_cached(q, ck, cv, table, keys, new, 1448), want)


def test_cached_of_any_int32(atlas):
    rng = np.random.default_rng(5)
    for new in ([1, 1], [40, 3]):
        keys = [130, 61]
        ck, cv, table, flat = paged(rng, keys, 2, 64, 16, 32)
        for spoil in ("q", "k", "v", "all"):
            k2, v2, q = ck.copy(), cv.copy(), values(rng, (sum(new), 4, 64))
            if spoil == "q":
                q[0, 1, 5] = -(1 << 31)
            if spoil == "k":
                k2[table[0, 3], 1, 2, 63] = (1 << 31) - 1
            if spoil == "v":
                v2[table[0, 3], 1, 2, 63] = (1 << 31) - 1
            if spoil == "all":
                q, k2, v2 = any_int32(rng, q.shape), any_int32(rng, ck.shape), any_int32(rng, cv.shape)
            assert np.array_equal(run_cached(q, k2, v2, table, keys, new, 2048), want_cached(q, k2, v2, table, flat, keys, new, 2048)), spoil
        c16 = rng.choice([-32768, 32767, 32640, 32639, 0], size=ck.shape).astype(np.int16)
        q = values(rng, (sum(new), 4, 64), 0.01)
        assert np.array_equal(run_cached(q, c16, c16, table, keys, new), want_cached(q, c16, c16, table, flat, keys, new))


@pytest.mark.parametrize("new", [1, 60, 700])
@pytest.mark.parametrize("causal", [True, False])
def test_a_table_without_columns(atlas, new, causal):
    """nothing can be cached: an empty table has no address, its rows are empty, and a step that needs a block does not fit"""
    import jolt_atlas_amd.attention as T
    rng = np.random.default_rng(new)
    at, cache = T.Attention(8, 2, 16, causal=causal), T.KVCache(*(Dev(np.zeros((3, 2, 16, 16), np.int32)) for _ in range(2)))
    q, out = Dev(values(rng, (new, 8, 16))), Dev(np.full((new, 8, 16), MARK, np.int32))
    table = Dev(np.zeros((1, 0), np.int32))
    table.data_ptr = lambda: 0
    at.cached(q, Dev(np.array([0, new], np.int32)), Dev(np.array([new], np.int32)), cache, table, out, workspace(at.cached_workspace_bytes(1, new, cache, 0)))
    assert not out.numpy().any()
    i32, pager = lambda *x: Dev(np.array(x, np.int32)), T.Pager(16, 3)  # noqa: E731
    for have, fresh, want in ((0, new, T.NO_COLUMNS), (0, 0, 0), (0, -1, 0)):
        status, cu, lens, n_out = i32(77), i32(77, 77), i32(77), i32(77)
        pager.plan(i32(have), i32(fresh), table, i32(0, 1, 2), i32(3), n_out, cu, lens, Dev(np.zeros(700, np.int64)), None, status, workspace(pager.workspace_bytes(1, 700)))
        assert (status.numpy()[0], n_out.numpy()[0], cu.numpy().tolist(), lens.numpy()[0]) == (want, 3, [0, 0], 0)


def test_rows_behind_the_last_sequence_stay(atlas):
    import jolt_atlas_amd.attention as T
    rng = np.random.default_rng(8)
    keys, new = [50, 20], [1, 1]
    ck, cv, table, flat = paged(rng, keys, 2, 16, 16, 32)
    q = values(rng, (6, 4, 16))
    at = T.Attention(4, 2, 16)
    cache = T.KVCache(Dev(ck), Dev(cv))
    out = Dev(np.full(q.shape, MARK, np.int32))
    at.cached(Dev(q), Dev(np.array([0, 1, 2], np.int32)), Dev(np.array(keys, np.int32)), cache, Dev(table), out, workspace(at.cached_workspace_bytes(2, 6, cache, table.shape[1])))
    got = out.numpy()
    assert (got[2:] == MARK).all() and np.array_equal(got[:2], want_cached(q[:2], ck, cv, table, flat, keys, new))


def test_cached_offsets_past_32_bits(atlas):
    """blocks whose elements lie beyond 2^32 elements of the cache: the allocation is never touched as a whole"""
    import jolt_atlas_amd.attention as T
    from _dev import Buffer
    rng = np.random.default_rng(13)
    KV, B, d = 8, 256, 256
    n_blocks = (1 << 32) // (KV * B * d) + 40
    size = n_blocks * KV * B * d
    bufs = [Buffer(2 * size) for _ in range(2)]
    one = values(rng, (2, KV, B, d), 0.4).clip(-32768, 32767).astype(np.int16)
    last = n_blocks - 1
    for b, x in zip(bufs, one):
        ok(hip().hipMemcpy(C.c_void_p(b.p.value + 2 * last * KV * B * d), np.ascontiguousarray(x).ctypes.data_as(C.c_void_p), C.c_size_t(x.nbytes), C.c_int(1)))
    views = []
    for b in bufs:
        v = Dev(np.empty(0, np.int16), b, 0, (n_blocks, KV, B, d), (KV * B * d, B * d, d, 1))
        v.total = 0
        views.append(v)
    cache = T.KVCache(*views)
    for new in (1, 40):
        at = T.Attention(KV, KV, d, 1024)
        q = values(rng, (new, KV, d))
        out = Dev(np.full(q.shape, MARK, np.int32))
        at.cached(Dev(q), Dev(np.array([0, new], np.int32)), Dev(np.array([200], np.int32)), cache, Dev(np.array([[last]], np.int32)), out, workspace(at.cached_workspace_bytes(1, new, cache, 1)))
        k, v = (x.transpose(1, 0, 2)[:200] for x in one)
        assert np.array_equal(out.numpy(), attend(q, k, v, [200 - new + j + 1 for j in range(new)], 1024))
    # and the write
    k, v = values(rng, (2, KV, d), 0.4), values(rng, (2, KV, d), 0.4)
    cache.write(Dev(k), Dev(v), Dev(np.array([last * B + 255, last * B], np.int64)))
    ok(hip().hipDeviceSynchronize())
    for b, x, was in zip(bufs, (k, v), one):
        got = np.empty((KV, B, d), np.int16)
        ok(hip().hipMemcpy(got.ctypes.data_as(C.c_void_p), C.c_void_p(b.p.value + 2 * last * KV * B * d), C.c_size_t(got.nbytes), C.c_int(2)))
        want = was.copy()
        want[:, 255], want[:, 0] = x[0].clip(-32768, 32767), x[1].clip(-32768, 32767)
        assert np.array_equal(got, want)


@pytest.mark.parametrize("H,KV,d,n,bits", [(2, 1, 64, 3000, 0), (2, 2, 128, 2500, 0), (1, 1, 32, 5000, 0), (3, 1, 200, 1500, 0), (1, 1, 16, 17000, 0), (2, 1, 128, 17000, 0), (4, 1, 64, 17001, 32),
                                           (2, 1, 256, 17001, 16), (16, 16, 64, 700, 0), (16, 8, 128, 500, 0)])
def test_long_sequences_on_some_of_their_rows(atlas, H, KV, d, n, bits):
    """many tiles, keys past what a tile holds e for; prompts (bits = 0) and chunks over a cache"""
    rng = np.random.default_rng(n)
    mul = int(round(ONE / np.sqrt(d)))
    new = n if bits == 0 else 150
    q, k, v = values(rng, (new, H, d)), values(rng, (n, KV, d)), values(rng, (n, KV, d))
    if bits == 0:
        got = run_prompt(atlas, q, k, v, [n], mul, pads=(0,))
    else:
        if bits == 16:
            k, v = (k // 8).clip(-32768, 32767), (v // 8).clip(-32768, 32767)
        B = 32
        up = -(-n // B)
        ids = rng.permutation(up).astype(np.int32)
        pages = np.zeros((2, up, KV, B, d), np.int16 if bits == 16 else np.int32)
        for c, x in zip(pages, (k, v)):
            c[ids] = np.concatenate([x, np.zeros((up * B - n, KV, d), np.int32)]).reshape(up, B, KV, d).transpose(0, 2, 1, 3)
        got = run_cached(q, pages[0], pages[1], ids[None], [n], [new], mul, caps=(0,))
    rows = sorted({0, 1, 31, 32, 63, new // 2, new - 1, *rng.integers(0, new, 6).tolist()})
    want = attend(q[rows], k, v, [n - new + r + 1 for r in rows], mul)
    assert np.array_equal(got[rows], want)


# ------------------------------------------------------------------------------------------------------------------- write
@pytest.mark.parametrize("d", [1, 4, 33, 64, 128, 255])
@pytest.mark.parametrize("bits", [32, 16])
@pytest.mark.parametrize("block", [1, 8, 64])
def test_write(atlas, d, bits, block):
    import jolt_atlas_amd.attention as T
    rng = np.random.default_rng(d)
    KV, n, n_blocks = 3, 50, 200 // block + 2
    dtype = np.int16 if bits == 16 else np.int32
    ck, cv = (rng.integers(-99, 99, size=(n_blocks, KV, block, d)).astype(dtype) for _ in range(2))
    wide = any_int32 if bits == 32 else (lambda r, s: r.integers(-32768, 32768, size=s).astype(np.int32))
    row = wide(rng, (n, 2 * KV, d + 3))
    R = Dev(row)
    k, v = (R.view(o * KV * (d + 3) + 1, (n, KV, d), (2 * KV * (d + 3), d + 3, 1)) for o in (0, 1))
    hk, hv = row[:, :KV, 1:d + 1], row[:, KV:, 1:d + 1]
    slots = rng.permutation(n_blocks * block)[:n].astype(np.int64)
    slots[[3, 17]] = [-1, -(1 << 40)]
    dk, dv, status = Dev(ck), Dev(cv), Dev(np.zeros(1, np.int32))
    cache = T.KVCache(dk, dv)
    cache.write(k, v, Dev(slots), status)
    cache.write(k, v, Dev(slots))
    for host, dev, src in ((ck, dk, hk), (cv, dv, hv)):
        want = host.copy()
        for i, s in enumerate(slots):
            if s >= 0:
                want[s // block, :, s % block] = src[i]
        assert np.array_equal(dev.numpy(), want)
    assert status.numpy()[0] == 0


def test_write_tells(atlas):
    import jolt_atlas_amd.attention as T
    ck = np.zeros((2, 1, 4, 5), np.int16)
    k = np.zeros((3, 1, 5), np.int32)
    k[1, 0, 4], k[2, 0, 0] = 40000, -(1 << 31)
    v = np.zeros((3, 1, 5), np.int32)
    dk, dv, status = Dev(ck), Dev(ck), Dev(np.zeros(1, np.int32))
    cache = T.KVCache(dk, dv)
    cache.write(Dev(k), Dev(v), Dev(np.array([0, 1, 7], np.int64)), status)
    assert status.numpy()[0] == T.NARROW
    got = dk.numpy()
    assert got[0, 0, 1, 4] == 32767 and got[1, 0, 3, 0] == -32768 and np.count_nonzero(got) == 2 and not dv.numpy().any()
    status = Dev(np.array([16], np.int32))
    cache.write(Dev(v), Dev(v), Dev(np.array([0, 8, 1 << 50], np.int64)), status)
    assert status.numpy()[0] == 16 | T.BAD_SLOT


# -------------------------------------------------------------------------------------------------------------------- plan
def run_plan(have, new, table, free, n_free, block, n_blocks, cap, positions=True):
    import jolt_atlas_amd.attention as T
    P = T.Pager(block, n_blocks)
    n = len(have)
    i32 = lambda x: Dev(np.asarray(x, np.int32))  # noqa: E731
    d = dict(table=Dev(table), free=Dev(free), n_free_out=i32([77]), cu=i32([77] * (n + 1)), lens=i32([77] * n), slots=Dev(np.full(cap, 77, np.int64)), positions=i32([77] * cap), status=i32([77]))
    P.plan(i32(have), i32(new), d["table"], d["free"], i32([n_free]), d["n_free_out"], d["cu"], d["lens"], d["slots"], d["positions"] if positions else None, d["status"],
           workspace(P.workspace_bytes(n, cap)))
    return {k: x.numpy() for k, x in d.items()}


def pool(rng, have, block, n_blocks, cols):
    ids = rng.permutation(n_blocks).astype(np.int32)
    table = np.full((len(have), cols), -1, np.int32)
    at = 0
    for i, c in enumerate(have):
        u = -(-c // block)
        table[i, :u] = ids[at:at + u]
        at += u
    free = np.full(n_blocks, -9, np.int32)
    free[:n_blocks - at] = ids[at:]
    return table, free, n_blocks - at


@pytest.mark.parametrize("n,longest,new,block,cap", [(1, 10, 1, 16, 1), (64, 500, 1, 64, 64), (64, 500, 1, 16, 100), (5, 0, 30, 8, 150), (1500, 60, 3, 4, 5000), (300, 40, 90, 16, 30000), (2500, 9, 1, 1, 2500),
                                                     (3, 4000, 5000, 4096, 15000)])
def test_plan(atlas, n, longest, new, block, cap):
    rng = np.random.default_rng(n)
    have = rng.integers(0, longest + 1, size=n)
    fresh = rng.integers(0, new + 1, size=n) if new > 1 else np.ones(n, int)
    fresh[rng.random(n) < 0.1] = -1
    cols = -(-(longest + new) // block) + 2
    n_blocks = int(sum(-(-(h + max(f, 0)) // block) for h, f in zip(have, fresh))) + 5
    table, free, n_free = pool(rng, have, block, n_blocks, cols)
    got = run_plan(have, fresh, table, free, n_free, block, n_blocks, cap)
    want = plan(list(have), list(fresh), table, free, n_free, block, n_blocks, cap)
    for k in want:
        assert np.array_equal(got[k], want[k]), k
    assert got["status"][0] == 0


@pytest.mark.parametrize("case", ["blocks", "columns", "tokens", "length", "ended_length", "stack", "stack_negative", "many_tokens", "exact_fit", "from_the_ended"])
def test_plan_that_does_not_fit_changes_nothing(atlas, case):
    rng = np.random.default_rng(1)
    have, new, block, n_blocks, cap, cols = [10, 3, 17, 0], [4, 1, -1, 20], 4, 40, 30, 10
    table, free, n_free = pool(rng, have, block, n_blocks, cols)
    if case == "blocks":
        free, n_free = np.full(n_blocks, 5, np.int32), 0
        new[2] = 0
    if case == "columns":
        table = np.ascontiguousarray(table[:, :4])
        have, new = [10, 3, 9, 0], [4, 1, -1, 20]
    if case == "tokens":
        cap = 24
    if case == "many_tokens":
        cap, new, cols = 5000, [4, 1, -1, 5000], 10
    if case == "length":
        have[1] = -1
    if case == "ended_length":
        new[0] = -2
    if case == "stack":
        n_free = n_blocks - 4
    if case == "stack_negative":
        n_free = -3
    if case == "exact_fit":
        cap, n_free, free = 25, 1, np.arange(n_blocks, dtype=np.int32)         # 5 given back + 1 = the 6 that are needed
    if case == "from_the_ended":
        n_free, new = 0, [2, 1, -1, 17]
    got = run_plan(have, new, table, free, n_free, block, n_blocks, cap)
    want = plan(have, new, table, free, n_free, block, n_blocks, cap)
    for k in want:
        assert np.array_equal(got[k], want[k]), (k, got[k], want[k])
    assert (want["status"][0] == 0) == (case in ("exact_fit", "from_the_ended"))


def test_plan_of_nothing(atlas):
    got = run_plan([], [], np.zeros((1, 2), np.int32), np.arange(4, dtype=np.int32), 4, 8, 4, 3, positions=False)
    assert got["status"][0] == 0 and got["cu"][0] == 0 and got["n_free_out"][0] == 4 and (got["slots"] == -1).all() and (got["positions"] == 77).all()


# ---------------------------------------------------------------------------------------------------- together, and the graph
def test_attention_is_the_traced_graphs(atlas):
    """atlas_graph_trace of the operator chain (the one atlas_prove_graph proves), and the operators over its q, k, v: the prompt at once, and token by token"""
    from jolt_atlas_amd import graph as GG
    from test_attention import chain
    import jolt_atlas_amd.attention as T
    for heads, seq, hd, mul in ((4, 64, 16, 4096), (16, 32, 64, 2048), (2, 128, 8, 5793)):
        nodes, q, k, v = chain(heads, seq, hd, seq, mul)
        G = GG.Graph(nodes, [nodes[-1]["idx"]])
        try:
            G.trace([q, k, v])
            want = G.node_output(nodes[-1]["idx"]).reshape(seq, heads, hd)
        finally:
            G.free()
        q, k, v = (x.reshape(seq, heads, hd) for x in (q, k, v))
        assert np.array_equal(run_prompt(atlas, q, k, v, [seq], mul), want)
        cache = T.KVCache(Dev(np.zeros((seq // 8, heads, 8, hd), np.int32)), Dev(np.zeros((seq // 8, heads, 8, hd), np.int32)))
        table = Dev(np.arange(seq // 8, dtype=np.int32)[::-1].reshape(1, -1).copy())
        at = T.Attention(heads, heads, hd, mul)
        ws = workspace(at.cached_workspace_bytes(1, 1, cache, seq // 8))
        for t in range(seq):
            slot = (seq // 8 - 1 - t // 8) * 8 + t % 8
            cache.write(Dev(k[t:t + 1]), Dev(v[t:t + 1]), Dev(np.array([slot], np.int64)))
            out = Dev(np.zeros((1, heads, hd), np.int32))
            at.cached(Dev(q[t:t + 1]), Dev(np.array([0, 1], np.int32)), Dev(np.array([t + 1], np.int32)), cache, table, out, ws)
            assert np.array_equal(out.numpy()[0], want[t]), t


def test_a_serving_run(atlas):
    """requests of different lengths through plan, write and cached attention over several steps — a prompt in one chunk, in pieces, token by token, one that ends
    and one that starts in its blocks — equal to attention over each whole sequence"""
    import jolt_atlas_amd.attention as T
    rng = np.random.default_rng(21)
    H, KV, d, B, n_blocks, cols, mul = 8, 2, 64, 8, 40, 16, 2048
    total = [70, 33, 50, 61]
    data = [tuple(values(rng, (t, h, d)) for h in (H, KV, KV)) for t in total]
    whole = [prompt(q, k, v, [len(q)], mul) for q, k, v in data]
    steps = [[40, 33, 0, 1], [1, -1, 7, 0], [1, 0, 20, 30], [28, 0, 1, 1], [0, 0, 22, 29]]
    at, pager = T.Attention(H, KV, d, mul), T.Pager(B, n_blocks)
    cap = 80
    cache = T.KVCache(Dev(rng.integers(-9, 9, (n_blocks, KV, B, d)).astype(np.int32)), Dev(rng.integers(-9, 9, (n_blocks, KV, B, d)).astype(np.int32)))
    i32 = lambda x: Dev(np.asarray(x, np.int32))  # noqa: E731
    table, free, n_free = i32(np.full((4, cols), -1)), i32(rng.permutation(n_blocks)), i32([n_blocks])
    cu, lens, slots, positions, status = i32([0] * 5), i32([0] * 4), Dev(np.zeros(cap, np.int64)), i32([0] * cap), i32([0])
    wp, wa = workspace(pager.workspace_bytes(4, cap)), workspace(at.cached_workspace_bytes(4, cap, cache, cols))
    have = [0] * 4
    for step in steps:
        pager.plan(i32(have), i32(step), table, free, n_free, n_free, cu, lens, slots, positions, status, wp)
        rows = [np.zeros((cap, h, d), np.int32) for h in (H, KV, KV)]
        at_row, want = 0, np.full((cap, H, d), MARK, np.int32)
        for i, f in enumerate(step):
            for x, src in zip(rows, data[i]):
                x[at_row:at_row + max(f, 0)] = src[have[i]:have[i] + max(f, 0)]
            want[at_row:at_row + max(f, 0)] = whole[i][have[i]:have[i] + max(f, 0)]
            at_row += max(f, 0)
            have[i] = 0 if f < 0 else have[i] + f
        out = Dev(np.full((cap, H, d), MARK, np.int32))
        cache.write(Dev(rows[1]), Dev(rows[2]), slots)
        at.cached(Dev(rows[0]), cu, lens, cache, table, out, wa)
        assert status.numpy()[0] == 0 and list(lens.numpy()) == have
        assert np.array_equal(out.numpy(), want)
    assert n_free.numpy()[0] == n_blocks - sum(-(-h // B) for h in have)


@pytest.mark.parametrize("cu", [[0, 40, 10, 60], [50, 20, 60, 0], [-5, 30, 60, 60], [0, 70, 80, 90], [2 ** 31 - 1, -(2 ** 31), 2 ** 31 - 1, 0], [0, 60, 0, 60]])
def test_offsets_that_make_no_sense_stay_inside(atlas, cu):
    """offsets that do not ascend, or pass the arrays: whatever is computed, nothing is written outside of out's rows and the workspace"""
    import jolt_atlas_amd.attention as T
    rng = np.random.default_rng(2)
    n, H, KV, d = 60, 4, 2, 64
    at = T.Attention(H, KV, d, 2048)
    big = Dev(np.full((n + 200, H, d), MARK, np.int32))
    out = big.view(100 * H * d, (n, H, d), (H * d, d, 1))
    q, k = Dev(values(rng, (n, H, d))), Dev(values(rng, (n, KV, d)))
    c = Dev(np.array(cu, np.int32))

    def guarded(size):
        w = workspace(size + 8192)
        return w, w.view(4096, (size,), (1,))

    def intact(w, size):
        x = w.numpy()
        assert (x[:4096] == 0xA5).all() and (x[4096 + size:] == 0xA5).all()
        y = big.numpy()
        assert (y[:100] == MARK).all() and (y[100 + n:] == MARK).all()

    size = at.prompt_workspace_bytes(3, n)
    w, v = guarded(size)
    at.prompt(q, k, k, c, out, v)
    intact(w, size)
    for rows, cols in ((n, 4), (n, 80), (n, 300)):
        ck = values(rng, (6, KV, 16, d))
        cache = T.KVCache(Dev(ck), Dev(ck))
        table = Dev(rng.integers(-2, 8, size=(3, cols)).astype(np.int32))
        size = at.cached_workspace_bytes(3, n, cache, cols)
        w, v = guarded(size)
        for lens in ([60, 60, 60], [cols * 16, -1, 2 ** 31 - 1]):
            at.cached(q, c, Dev(np.array(lens, np.int32)), cache, table, out, v)
            intact(w, size)


@pytest.mark.parametrize("H,KV,d", [(4, 2, 64), (8, 1, 128), (2, 2, 256), (6, 2, 36), (40, 1, 16)])
@pytest.mark.parametrize("cu", [[0, 60, 60, 101], [0, 2, 3, 4], [0, 101, 30, 101], [101, 0, 101, 7]])
def test_a_call_stays_inside_what_it_needs(atlas, H, KV, d, cu):
    """a workspace may be smaller than the size functions' (they cover smaller calls too), down to what the call's own path needs: no byte behind that is touched"""
    import jolt_atlas_amd.attention as T
    rng = np.random.default_rng(d)
    at = T.Attention(H, KV, d, 2048)
    c = Dev(np.array(cu, np.int32))

    def least(call, most):
        lo, hi = 0, most                         # the smallest that is not refused
        while lo < hi:
            mid = (lo + hi) // 2
            try:
                call(Dev(np.empty(0, np.uint8), whole, 4096, (mid,), (1,)))
                hi = mid
            except atlas.AtlasError as e:
                assert "workspace" in str(e)
                lo = mid + 1
        return lo

    def check(call, most):
        nonlocal whole
        w = workspace(most + 8192)
        whole = w.buf
        size = least(call, most)
        assert 0 < size <= most
        ok(hip().hipDeviceSynchronize())
        w = workspace(size + 8192)
        call(w.view(4096, (size,), (1,)))
        x = w.numpy()
        assert (x[:4096] == 0xA5).all() and (x[4096 + size:] == 0xA5).all()

    whole = None
    for rows in (101, 2100, 16500):
        q, k, out = (Dev(np.zeros((rows, h, d), np.int32)) for h in (H, KV, H))
        check(lambda ws: at.prompt(q, k, k, c, out, ws), at.prompt_workspace_bytes(3, rows))
    ck = values(rng, (6, KV, 16, d))
    cache = T.KVCache(Dev(ck), Dev(ck))
    for rows in (4, 101):
        q, out = (Dev(np.zeros((rows, H, d), np.int32)) for _ in range(2))
        for cols in (4, 80, 300, 1040):
            table, lens = Dev(rng.integers(-2, 8, size=(3, cols)).astype(np.int32)), Dev(np.array([cols * 16, 70, 2 ** 31 - 1], np.int32))
            check(lambda ws: at.cached(q, c, lens, cache, table, out, ws), at.cached_workspace_bytes(3, rows, cache, cols))


@pytest.mark.parametrize("d", [32, 128])
def test_every_kernel_captured(atlas, d):
    """tiles, tiles of long sequences and the split path inside one graph, replayed over changed inputs"""
    import jolt_atlas_amd.attention as T
    h = hip()
    rng = np.random.default_rng(d)
    H, KV, n, B = 4, 2, 40, 16
    at = T.Attention(H, KV, d, 2048)
    st, graph, exe = C.c_void_p(), C.c_void_p(), C.c_void_p()
    ok(h.hipStreamCreateWithFlags(C.byref(st), C.c_uint(1)))
    rows = 16500
    q, k, v = (Dev(np.zeros((rows, x, d), np.int32)) for x in (H, KV, KV))
    outs = [Dev(np.zeros((rows, H, d), np.int32)) for _ in range(4)]
    cu = Dev(np.array([0, 25, n], np.int32))
    ck, cv, table, flat = paged(rng, [70, 30], KV, d, B, 32)
    cache, cq, one = T.KVCache(Dev(ck), Dev(cv)), Dev(np.zeros((2, H, d), np.int32)), Dev(np.array([0, 1, 2], np.int32))
    lens, wide = Dev(np.array([70, 30], np.int32)), Dev(np.concatenate([table, np.full((2, 300), -1, np.int32)], axis=1))
    calls = []
    for x, m in zip(outs, (n, 2100, rows)):
        cut = lambda y: y.view(0, (m,) + y.shape[1:], y.stride())  # noqa: E731
        calls.append(lambda s, a=(cut(q), cut(k), cut(v), cu, cut(x), workspace(at.prompt_workspace_bytes(2, m))): at.prompt(*a, stream=s))
    cout = outs[3].view(0, (2, H, d), (H * d, d, 1))
    cws = workspace(at.cached_workspace_bytes(2, 2, cache, wide.shape[1]))
    calls.append(lambda s: at.cached(cq, one, lens, cache, wide, cout, cws, stream=s))
    ok(h.hipDeviceSynchronize())
    ok(h.hipStreamBeginCapture(st, C.c_int(0)))
    for f in calls:
        f(st.value)
    ok(h.hipStreamEndCapture(st, C.byref(graph)))
    ok(h.hipGraphInstantiate(C.byref(exe), graph, None, None, C.c_size_t(0)))
    for rep in range(3):
        hq, hk, hv, hc = values(rng, (n, H, d)), values(rng, (n, KV, d)), values(rng, (n, KV, d)), values(rng, (2, H, d))
        for dev, x in ((q, hq), (k, hk), (v, hv), (cq, hc)):
            ok(h.hipMemcpy(dev.buf.p, np.ascontiguousarray(x).ctypes.data_as(C.c_void_p), C.c_size_t(x.nbytes), C.c_int(1)))
        ok(h.hipDeviceSynchronize())
        ok(h.hipGraphLaunch(exe, st))
        ok(h.hipDeviceSynchronize())
        want = prompt(hq, hk, hv, [25, 15], 2048)
        for x in outs[:3]:
            assert np.array_equal(x.numpy()[:n], want), rep
        assert np.array_equal(cout.numpy(), want_cached(hc, ck, cv, table, flat, [70, 30], [1, 1], 2048)), rep
        run_prompt(atlas, hq, hk, hv, [25, 15], 2048, pads=(2100,))          # eager work between the replays
    ok(h.hipGraphExecDestroy(exe))
    ok(h.hipGraphDestroy(graph))
    ok(h.hipStreamDestroy(st))


@pytest.mark.parametrize("cols", [16, 200])
def test_a_whole_step_captured(atlas, cols):
    """the plan, the write and the attention with its question about the mask in one graph, replayed step by step over new lengths, keys and queries"""
    import jolt_atlas_amd.attention as T
    h, rng = hip(), np.random.default_rng(cols)
    H, KV, d, B, n_blocks, cap, mul, fill = 4, 2, 64, 8, 60, 70, 2048, -(8 << 14)
    total = [100, 61, 90]
    data = [tuple(values(rng, (t, x, d), 0.6) for x in (H, KV, KV)) for t in total]
    whole = [prompt(q, k, v, [len(q)], mul) for q, k, v in data]
    at, pager = T.Attention(H, KV, d, mul, mask_fill=fill, mask_tokens=64), T.Pager(B, n_blocks)
    i32 = lambda x: Dev(np.asarray(x, np.int32))  # noqa: E731
    cache = T.KVCache(*(Dev(np.zeros((n_blocks, KV, B, d), np.int32)) for _ in range(2)))
    have, new, table, free, n_free = i32([0] * 3), i32([0] * 3), i32(np.full((3, cols), -1)), i32(rng.permutation(n_blocks)), i32([n_blocks])
    cu, lens, slots, positions, status, told, narrow = i32([0] * 4), i32([0] * 3), Dev(np.zeros(cap, np.int64)), i32([0] * cap), i32([0]), i32([0]), i32([0])
    rows, out = [Dev(np.zeros((cap, x, d), np.int32)) for x in (H, KV, KV)], Dev(np.zeros((cap, H, d), np.int32))
    wp, wa = workspace(pager.workspace_bytes(3, cap)), workspace(at.cached_workspace_bytes(3, cap, cache, cols))
    up = lambda dev, x: ok(h.hipMemcpy(dev.buf.p, np.ascontiguousarray(x).ctypes.data_as(C.c_void_p), C.c_size_t(x.nbytes), C.c_int(1)))  # noqa: E731
    st, graph, exe = C.c_void_p(), C.c_void_p(), C.c_void_p()
    ok(h.hipStreamCreateWithFlags(C.byref(st), C.c_uint(1)))
    ok(h.hipDeviceSynchronize())
    ok(h.hipStreamBeginCapture(st, C.c_int(0)))
    pager.plan(have, new, table, free, n_free, n_free, cu, lens, slots, positions, status, wp, stream=st.value)
    cache.write(rows[1], rows[2], slots, narrow, stream=st.value)
    at.cached(rows[0], cu, lens, cache, table, out, wa, stream=st.value, status=told)
    ok(h.hipStreamEndCapture(st, C.byref(graph)))
    ok(h.hipGraphInstantiate(C.byref(exe), graph, None, None, C.c_size_t(0)))
    now, seen = [0] * 3, set()
    for step in ([20, 0, 1], [1, 1, 1], [30, 10, 29], [0, 50, 1], [1, -1, 1], [48, 0, 22], [0, 0, 0], [0, 61, 9]):
        hrows, want, first, expect = [np.zeros((cap, x, d), np.int32) for x in (H, KV, KV)], np.full((cap, H, d), MARK, np.int32), 0, False
        for i, f in enumerate(step):
            if f < 0:
                now[i] = 0
                continue
            for x, src in zip(hrows, data[i]):
                x[first:first + f] = src[now[i]:now[i] + f]
            want[first:first + f] = whole[i][now[i]:now[i] + f]
            q, k, _ = data[i]
            expect |= mask_weighs(q[now[i]:now[i] + f], k, list(range(now[i] + 1, now[i] + f + 1)), list(range(now[i], now[i] + f)), mul, fill, 64)
            now[i] += f
            first += f
        had = lens.numpy()                       # a request that ends brings the tokens it has
        up(have, np.array([had[i] if f < 0 else now[i] - f for i, f in enumerate(step)], np.int32))
        up(new, np.array(step, np.int32))
        for dev, x in zip(rows, hrows):
            up(dev, x)
        up(out, np.full((cap, H, d), MARK, np.int32))
        up(told, np.zeros(1, np.int32))
        ok(h.hipDeviceSynchronize())
        ok(h.hipGraphLaunch(exe, st))
        ok(h.hipDeviceSynchronize())
        assert status.numpy()[0] == 0 and narrow.numpy()[0] == 0 and lens.numpy().tolist() == now
        assert np.array_equal(out.numpy(), want), step
        assert told.numpy()[0] == (T.MASK_WEIGHS if expect else 0), step
        seen.add(expect)
        assert n_free.numpy()[0] == n_blocks - sum(-(-n // B) for n in now)
        x = values(rng, (30, H, d)), values(rng, (30, KV, d)), values(rng, (30, KV, d))          # eager work between the replays
        assert np.array_equal(run_prompt(atlas, *x, [30], mul, pads=(0,)), prompt(*x, [30], mul))
    assert seen == {False, True}
    ok(h.hipGraphExecDestroy(exe))
    ok(h.hipGraphDestroy(graph))
    ok(h.hipStreamDestroy(st))


def test_pointers_that_are_no_device_memory(atlas):
    import jolt_atlas_amd.attention as T
    at = T.Attention(1, 1, 4)
    x = Dev(np.zeros((2, 1, 4), np.int32))
    host = np.zeros((2, 1, 4), np.int32)
    fake = Dev(np.empty(0, np.int32), x.buf, 0, (2, 1, 4), (4, 4, 1))
    fake.data_ptr = lambda: host.ctypes.data
    y = Dev(host)
    for a in ((fake, x, x, y), (x, fake, x, y), (x, x, fake, y), (x, x, x, fake)):
        with pytest.raises(atlas.AtlasError, match="device"):
            at.prompt(a[0], a[1], a[2], Dev(np.array([0, 2], np.int32)), a[3], workspace(at.prompt_workspace_bytes(1, 2)))


def test_captured_and_replayed_on_two_streams(atlas):
    """a step captured into two graphs on two streams (a workspace each), replayed over changed inputs, with eager calls between; each replay against the definition"""
    import jolt_atlas_amd.attention as T
    h = hip()
    rng = np.random.default_rng(4)
    H, KV, d, B = 4, 2, 64, 16
    up = lambda dev, x: ok(h.hipMemcpy(dev.buf.p, np.ascontiguousarray(x).ctypes.data_as(C.c_void_p), C.c_size_t(x.nbytes), C.c_int(1)))  # noqa: E731
    sides = []
    for side in range(2):
        keys, new = ([300, 41], [1, 1]) if side == 0 else ([90, 130], [20, 3])
        ck, cv, table, flat = paged(rng, keys, KV, d, B, 32)
        S = dict(keys=keys, new=new, table=table, ck=ck, cv=cv, flat=flat, at=T.Attention(H, KV, d, 2048), q=Dev(np.zeros((sum(new), H, d), np.int32)), k=Dev(np.zeros((sum(new), KV, d), np.int32)),
                 v=Dev(np.zeros((sum(new), KV, d), np.int32)), out=Dev(np.zeros((sum(new), H, d), np.int32)), pout=Dev(np.zeros((sum(new), H, d), np.int32)), cache=T.KVCache(Dev(ck), Dev(cv)))
        S["lens"], S["cu"], S["dtable"] = Dev(np.array(keys, np.int32)), Dev(np.cumsum([0] + new).astype(np.int32)), Dev(table)
        slots = []
        for i, (m, n) in enumerate(zip(keys, new)):
            slots += [int(table[i, p // B]) * B + p % B for p in range(m - n, m)]
        S["slots"], S["hslots"] = Dev(np.array(slots, np.int64)), slots
        S["ws"] = workspace(S["at"].cached_workspace_bytes(2, sum(new), S["cache"], table.shape[1]))
        S["pws"] = workspace(S["at"].prompt_workspace_bytes(2, sum(new)))
        S["stream"] = C.c_void_p()
        ok(h.hipStreamCreateWithFlags(C.byref(S["stream"]), C.c_uint(1)))
        ok(h.hipDeviceSynchronize())
        graph, S["exec"] = C.c_void_p(), C.c_void_p()
        ok(h.hipStreamBeginCapture(S["stream"], C.c_int(0)))
        step(S, S["stream"].value)
        ok(h.hipStreamEndCapture(S["stream"], C.byref(graph)))
        ok(h.hipGraphInstantiate(C.byref(S["exec"]), graph, None, None, C.c_size_t(0)))
        ok(h.hipGraphDestroy(graph))
        sides.append(S)
    for rep in range(4):
        for S in sides:
            S["hq"], S["hk"], S["hv"] = values(rng, S["q"].shape), values(rng, S["k"].shape), values(rng, S["v"].shape)
            up(S["q"], S["hq"]), up(S["k"], S["hk"]), up(S["v"], S["hv"])
        ok(h.hipDeviceSynchronize())
        for S in sides:
            ok(h.hipGraphLaunch(S["exec"], S["stream"]))
        if rep % 2:                          # eager work of the program's own, on the library stream, between the replays
            x = values(rng, (40, H, d)), values(rng, (40, KV, d)), values(rng, (40, KV, d))
            assert np.array_equal(run_prompt(atlas, *x, [40], 2048), prompt(*x, [40], 2048))
        ok(h.hipDeviceSynchronize())
        for S in sides:
            for i, s in enumerate(S["hslots"]):
                S["ck"][s // B, :, s % B], S["cv"][s // B, :, s % B] = S["hk"][i], S["hv"][i]
            assert np.array_equal(S["out"].numpy(), want_cached(S["hq"], S["ck"], S["cv"], S["table"], S["flat"], S["keys"], S["new"], 2048)), rep
            assert np.array_equal(S["pout"].numpy(), prompt(S["hq"], S["hk"], S["hv"], S["new"], 2048)), rep
    for S in sides:
        step(S, 0)                           # HIP's default stream
        assert np.array_equal(S["pout"].numpy(), prompt(S["hq"], S["hk"], S["hv"], S["new"], 2048))
        ok(h.hipGraphExecDestroy(S["exec"]))
        ok(h.hipStreamDestroy(S["stream"]))


def step(S, stream):
    S["cache"].write(S["k"], S["v"], S["slots"], stream=stream)
    S["at"].cached(S["q"], S["cu"], S["lens"], S["cache"], S["dtable"], S["out"], S["ws"], stream=stream)
    S["at"].prompt(S["q"], S["k"], S["v"], S["cu"], S["pout"], S["pws"], stream=stream)


def test_calls_of_two_threads(atlas):
    """two threads that share the runtime, each with its own stream and workspace, at once"""
    import threading
    import jolt_atlas_amd.attention as T
    h, wrong = hip(), []

    def work(seed):
        rng = np.random.default_rng(seed)
        st = C.c_void_p()
        ok(h.hipSetDevice(C.c_int(0)))
        ok(h.hipStreamCreateWithFlags(C.byref(st), C.c_uint(1)))
        at = T.Attention(4, 2, 64, 2048)
        q, k, v = values(rng, (90, 4, 64)), values(rng, (90, 2, 64)), values(rng, (90, 2, 64))
        want = prompt(q, k, v, [50, 40], 2048)
        dev, ws, cu = [Dev(x) for x in (q, k, v)], workspace(at.prompt_workspace_bytes(2, 90)), Dev(np.array([0, 50, 90], np.int32))
        for _ in range(20):
            out = Dev(np.zeros(q.shape, np.int32))
            at.prompt(*dev, cu, out, ws, stream=st.value)
            ok(h.hipStreamSynchronize(st))
            if not np.array_equal(out.numpy(), want):
                wrong.append(seed)
        ok(h.hipStreamDestroy(st))

    threads = [threading.Thread(target=work, args=(s,)) for s in (1, 2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


def test_calls_of_two_threads_of_other_sizes(atlas):
    """the scores of a short prompt stay in LDS: threads whose prompts need more and less of it do not take it from each other"""
    import threading
    import jolt_atlas_amd.attention as T
    h, wrong = hip(), []
    rng = np.random.default_rng(6)
    start = threading.Barrier(4)

    def work(rows):
        try:
            st = C.c_void_p()
            ok(h.hipSetDevice(C.c_int(0)))
            ok(h.hipStreamCreateWithFlags(C.byref(st), C.c_uint(1)))
            at = T.Attention(1, 1, 64, 2048)
            x, out, cu, ws = Dev(np.zeros((rows, 1, 64), np.int32)), Dev(np.zeros((rows, 1, 64), np.int32)), Dev(np.array([0, 3], np.int32)), workspace(at.prompt_workspace_bytes(1, rows))
            start.wait()
            for _ in range(1500):
                at.prompt(x, x, x, cu, out, ws, stream=st.value)
            ok(h.hipStreamSynchronize(st))
            ok(h.hipStreamDestroy(st))
        except Exception as e:  # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(n,)) for n in (2000, 1000, 1990, 1010)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong, wrong


def test_an_error_that_the_caller_left(atlas):
    """an earlier HIP call of the caller's failed: that is not the attention's error"""
    import jolt_atlas_amd.attention as T
    h, rng = hip(), np.random.default_rng(3)
    at, pager = T.Attention(1, 1, 8), T.Pager(4, 8)
    q, k, v = (values(rng, (5, 1, 8)) for _ in range(3))
    dev, out, cu, ws = [Dev(x) for x in (q, k, v)], Dev(np.zeros((5, 1, 8), np.int32)), Dev(np.array([0, 5], np.int32)), workspace(at.prompt_workspace_bytes(1, 5))
    i32 = lambda *x: Dev(np.array(x, np.int32))  # noqa: E731
    cache, ck, slots = T.KVCache(Dev(np.zeros((8, 1, 4, 8), np.int32)), Dev(np.zeros((8, 1, 4, 8), np.int32))), Dev(np.zeros((5, 1, 8), np.int32)), Dev(np.zeros(5, np.int64))
    have, new, table, free, n_free, lens, status = i32(0), i32(5), i32(0, 0).view(0, (1, 2), (2, 1)), i32(*range(8)), i32(8), i32(0), i32(7)
    wp, wc, pcu = workspace(pager.workspace_bytes(1, 5)), workspace(at.cached_workspace_bytes(1, 5, cache, 2)), i32(0, 0)
    calls = [lambda: at.prompt(*dev, cu, out, ws), lambda: pager.plan(have, new, table, free, n_free, n_free, pcu, lens, slots, None, status, wp),
             lambda: cache.write(dev[1], dev[2], slots), lambda: at.cached(dev[0], pcu, lens, cache, table, ck, wc)]
    for f in calls:
        assert h.hipSetDevice(C.c_int(4096)) != 0
        f()
    want = prompt(q, k, v, [5])
    assert status.numpy()[0] == 0 and np.array_equal(out.numpy(), want) and np.array_equal(ck.numpy(), want)


def masked_status(q, k, v, lens, mul, fill, tokens, steps, want):
    """the status of a prompt and of the same rows over a cache (in `steps` new tokens each), through every kernel; both outputs are `want`"""
    import jolt_atlas_amd.attention as T
    n, H, d = q.shape
    KV, B = k.shape[1], 16
    at, plain, told = T.Attention(H, KV, d, mul, mask_fill=fill, mask_tokens=tokens), T.Attention(H, KV, d, mul), set()
    word = lambda: Dev(np.array([1 << 30], np.uint32))  # noqa: E731
    for rows in (n, 2100, 16500):
        more = lambda x: Dev(np.concatenate([x, np.full((rows - n,) + x.shape[1:], 1 << 20, np.int32)]))  # noqa: E731
        a = (more(q), more(k), more(v), Dev(np.cumsum([0] + lens).astype(np.int32)), Dev(np.zeros((rows, H, d), np.int32)), workspace(at.prompt_workspace_bytes(len(lens), rows)))
        st = word()
        assert np.array_equal(at.prompt(*a, status=st).numpy()[:n], want) and np.array_equal(plain.prompt(*a).numpy()[:n], want)
        told.add(int(st.numpy()[0]))
    up = [-(-x // B) for x in lens]
    ck, cv = (np.zeros((sum(up) + 1, KV, B, d), np.int32) for _ in range(2))
    table, base, first = np.full((len(lens), max(up)), -1, np.int32), 1, 0
    for i, x in enumerate(lens):
        table[i, :up[i]] = base + np.arange(up[i])
        for c, src in ((ck, k), (cv, v)):
            flat = np.zeros((up[i] * B, KV, d), np.int32)
            flat[:x] = src[first:first + x]
            c[base:base + up[i]] = flat.reshape(up[i], B, KV, d).transpose(0, 2, 1, 3)
        base += up[i]
        first += x
    cache, at_row = T.KVCache(Dev(ck), Dev(cv)), np.cumsum([0] + lens)
    for cols in (max(up), 70, 263, 1040):
        wide, st, got = Dev(np.concatenate([table, np.full((len(lens), cols - max(up)), -1, np.int32)], axis=1)), word(), np.zeros_like(q)
        for p in range(0, max(lens), steps):
            new = [max(0, min(steps, x - p)) for x in lens]
            sel = np.concatenate([at_row[i] + p + np.arange(m) for i, m in enumerate(new)]).astype(int)
            out = Dev(np.zeros((len(sel), H, d), np.int32))
            a = (Dev(q[sel]), Dev(np.cumsum([0] + new).astype(np.int32)), Dev(np.array([min(x, p + m) for x, m in zip(lens, new)], np.int32)), cache, wide, out,
                 workspace(at.cached_workspace_bytes(len(lens), len(sel), cache, cols)))
            got[sel] = at.cached(*a, status=st).numpy()
            assert np.array_equal(plain.cached(*a).numpy(), got[sel])
        assert np.array_equal(got, want), cols
        told.add(int(st.numpy()[0]))
    assert len(told) == 1 and told <= {1 << 30, 1 << 30 | T.MASK_WEIGHS}, told
    return told == {1 << 30 | T.MASK_WEIGHS}


def status_of(q, k, lens, mul, fill, tokens):
    at = np.cumsum([0] + list(lens))
    return any(mask_weighs(q[a:b], k[a:b], list(range(1, b - a + 1)), list(range(b - a)), mul, fill, tokens) for a, b in zip(at, at[1:]))


@pytest.mark.parametrize("H,KV,d,steps", [(2, 1, 16, 9), (4, 2, 64, 1), (2, 2, 128, 40), (3, 1, 33, 40), (8, 1, 256, 7), (2, 1, 200, 40)])
@pytest.mark.parametrize("spoil", [None, "q", "v"])
def test_a_mask_that_would_weigh(atlas, H, KV, d, steps, spoil):
    """fills around every border of e: where it is 0, where it is 1 between zeros, the maximum itself, above; some of it in rows of operands of any size"""
    rng = np.random.default_rng(d)
    lens = [40, 1, 23]
    n = sum(lens)
    q, k, v = values(rng, (n, H, d), 0.5), values(rng, (n, KV, d), 0.5), values(rng, (n, KV, d))
    if spoil == "q":
        q[n - 5, 0, 0] = -(1 << 31)
    if spoil == "v":
        v[17, 0, d - 1] = (1 << 31) - 1
    mul = int(round(ONE / np.sqrt(d)))
    want = prompt(q, k, v, lens, mul)
    # the least maximum of a row that has masked keys: the lowest fill that would be it
    lo, hi = -(1 << 31), (1 << 31) - 1
    while lo < hi:
        mid = (lo + hi) // 2
        if any(mask_weighs(q[a:a + m], k[a:a + m], list(range(1, m + 1)), list(range(m)), mul, mid, 64) for a, m in zip(np.cumsum([0] + lens), lens)):
            hi = mid
        else:
            lo = mid + 1
    seen = set()
    for fill in (lo - 1, lo, lo + 511, lo + (1 << 18), -(1 << 31), (1 << 31) - 1):
        expect = status_of(q, k, lens, mul, fill, 64)
        seen.add(expect)
        assert masked_status(q, k, v, lens, mul, fill, 64, steps, want) == expect, fill
    assert seen == {False, True}
    assert not masked_status(q, k, v, lens, mul, (1 << 31) - 1, 1, steps, want)                # a graph of one token has no masked keys


@pytest.mark.parametrize("tokens", [23, 24, 39, 40, 41, 64])
def test_the_last_token_of_a_graph_has_no_masked_keys(atlas, tokens):
    rng = np.random.default_rng(tokens)
    lens, mul = [40, 23], 2048
    q, k, v = (values(rng, (63, h, 64)) for h in (4, 2, 2))
    q[:39], q[40:] = k[:39].repeat(2, axis=1), k[40:].repeat(2, axis=1)                        # all rows high, but the 40th token of one sequence
    q[39] = -k[:40].sum(axis=0, dtype=np.int64).clip(-(1 << 17), 1 << 17).repeat(2, axis=0).astype(np.int32)
    want = prompt(q, k, v, lens, mul)
    for fill in (-(10 << 14), 0, 1 << 20):
        assert masked_status(q, k, v, lens, mul, fill, tokens, 8, want) == status_of(q, k, lens, mul, fill, tokens)


@pytest.mark.parametrize("name,weighs", [("microgpt_model", False), ("nanogpt_model", False), ("nanogpt", True), ("gpt2_layer", True)])
def test_attention_of_the_frameworks_graphs(atlas, name, weighs):
    """the layers of the framework's own graphs, their fill -10 or -8: equal to the trace where the status stays clear, and told where it does not"""
    from test_attention import graph_attention
    told = False
    for (q, k, v), mul, fill, trace in graph_attention(name):
        n = len(q)
        want = prompt(q, k, v, [n], mul)
        tell = masked_status(q, k, v, [n], mul, fill, n, 5, want)
        assert tell == status_of(q, k, [n], mul, fill, n)
        assert tell or np.array_equal(want, trace)
        told |= tell
    assert told == weighs


TORCH = """
import sys
import torch
sys.path[:0] = [ROOT, ROOT + "/tests"]
import jolt_atlas_amd as A
import jolt_atlas_amd.attention as T
import numpy as np
from _attention_ref import prompt
A.init(0)
g = torch.Generator().manual_seed(5)
n, H, KV, d, B = 90, 4, 2, 64, 16
at = T.Attention(H, KV, d, 2048)
cu = torch.tensor([0, 50, 90], dtype=torch.int32, device="cuda")
ws = torch.empty(at.prompt_workspace_bytes(2, n), dtype=torch.uint8, device="cuda")
big = torch.zeros(1 << 28, device="cuda")
for side in (None, torch.cuda.Stream()):
    with torch.cuda.stream(side or torch.cuda.default_stream()):
        for rep in range(3):
            h = [(torch.randn(n, x, d, generator=g) * 16384).round().to(torch.int32) for x in (H, KV, KV)]
            q, k, v = (torch.zeros_like(x, device="cuda") for x in h)
            out, src = torch.zeros_like(q), [x.pin_memory() for x in h]
            torch.cuda.synchronize()
            for _ in range(40):
                big.add_(1.0)                          # some 20 ms of work: q, k and v come behind it
            for x, y in zip((q, k, v), src):
                x.copy_(y, non_blocking=True)
            at.prompt(q, k, v, cu, out, ws)
            kept = out.clone()                         # torch's next operation comes behind the call
            out.zero_()
            assert np.array_equal(kept.cpu().numpy(), prompt(*(x.numpy() for x in h), [50, 40], 2048)), (side, rep)
            cache = T.KVCache(*(torch.zeros(9, KV, B, d, dtype=torch.int32, device="cuda") for _ in range(2)))
            i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
            pager, table, free = T.Pager(B, 9), i32(*[-1] * 8).reshape(2, 4), i32(*range(9))
            have, cun, lens, n_free = i32(0, 0), i32(0, 0, 0), i32(0, 0), i32(9)
            slots, status = torch.zeros(100, dtype=torch.int64, device="cuda"), i32(7)
            wp = torch.empty(pager.workspace_bytes(2, 100), dtype=torch.uint8, device="cuda")
            pager.plan(have, i32(50, 40), table, free, n_free, n_free, cun, lens, slots, None, status, wp)
            cache.write(k, v, slots, status)
            out = torch.zeros_like(q)
            wc = torch.empty(at.cached_workspace_bytes(2, n, cache, 4), dtype=torch.uint8, device="cuda")
            at.cached(q, cun, lens, cache, table, out, wc)
            assert int(status) == 0 and torch.equal(out, kept), (side, rep, int(status))
print("torch ok", flush=True)
"""


def test_torch_tensors(tmp_path):
    """torch tensors on torch's current stream, in a process of their own (torch comes first there)"""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    f = tmp_path / "run.py"
    f.write_text("ROOT = %r\n%s" % (root, TORCH))
    r = subprocess.run([sys.executable, "-u", str(f)], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "torch ok" in r.stdout, r.stdout + r.stderr
