"""CPU: the exp tables compiled into the attention kernels are the graph executor's, and every refusal of the attention and paging entry points answers on
the host before anything touches a device."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_exp_tables_are_the_graph_executors(tmp_path):
    from _attention_ref import exp_tables
    src = tmp_path / "t.cpp"
    src.write_text('#include "%s/jolt-atlas_amd/csrc/exp_table.hpp"\n#include <cstdio>\nint main() { constexpr auto t = atlas::make_exp_table();\n'
                   'for (int v : t.hi) printf("%%d\\n", v);\nfor (int v : t.lo) printf("%%d\\n", v);\n}' % ROOT)
    subprocess.check_call(["g++", "-std=c++17", str(src), "-o", str(tmp_path / "t")])
    got = np.array([int(x) for x in subprocess.check_output([str(tmp_path / "t")], text=True).split()])
    hi, lo = exp_tables()
    assert np.array_equal(got[:512], hi) and np.array_equal(got[512:], lo)


def test_the_reference_is_the_graph_operators():
    """tests/_attention_ref.py against the oracle executor's operator chain: Einsum, Mul, Iff, SoftmaxLastAxis, Einsum"""
    from _attention_ref import prompt
    from oracle import graph as OG
    nodes, q, k, v = chain(4, 16, 8, 3, 2896)
    out, _ = OG.execute(nodes, [q, k, v])
    got = prompt(q.reshape(16, 4, 8), k.reshape(16, 4, 8), v.reshape(16, 4, 8), [16], 2896)
    assert np.array_equal(out[nodes[-1]["idx"]].reshape(16, 4, 8), got)


def chain(heads, seq, hd, seed, score_mul, sigma=1.0):
    """the attention of a model graph, its mask filled far below every score"""
    rng = np.random.default_rng(seed)
    q, k, v = (np.clip(np.round(rng.normal(0, sigma * (1 << 14), seq * heads * hd)), -(1 << 18), (1 << 18) - 1).astype(np.int32) for _ in range(3))
    full = lambda x: np.full(heads * seq * seq, x, dtype=np.int32)  # noqa: E731
    mask = np.broadcast_to(np.tril(np.ones((seq, seq), np.int32)), (heads, seq, seq)).reshape(-1)
    dims = [heads, seq, seq]
    nodes = [{"op": "Input", "inputs": [], "dims": [seq, heads, hd]}] * 3 + [
        {"op": "Einsum", "inputs": [0, 1], "dims": dims, "layout": "mbk,nbk->bmn", "scale": 14, "shape": [heads, seq, hd, seq]},
        {"op": "Constant", "inputs": [], "dims": dims, "data": full(score_mul)},
        {"op": "Mul", "inputs": [3, 4], "dims": dims, "scale": 14},
        {"op": "Constant", "inputs": [], "dims": dims, "data": mask},
        {"op": "Constant", "inputs": [], "dims": dims, "data": full(-(1 << 27))},
        {"op": "Iff", "inputs": [6, 5, 7], "dims": dims},
        {"op": "SoftmaxLastAxis", "inputs": [8], "dims": dims, "scale": 14},
        {"op": "Einsum", "inputs": [9, 2], "dims": [seq, heads, hd], "layout": "bmk,kbn->mbn", "scale": 14, "shape": [heads, seq, seq, hd]}]
    return [dict(nd, idx=i) for i, nd in enumerate(nodes)], q, k, v


class Fake:
    """a tensor's shape with an address that nothing may look at"""

    def __init__(self, shape, dtype="int32", strides=None, ptr=1 << 40):
        self.shape, self.dtype, self.ptr = tuple(shape), np.dtype(dtype), ptr
        self.itemsize = self.dtype.itemsize
        self._s = tuple(strides) if strides else tuple(int(np.prod(shape[i + 1:])) for i in range(len(shape)))

    def data_ptr(self):
        return self.ptr

    def stride(self):
        return self._s


def _prompt(**kw):
    import jolt_atlas_amd.attention as T
    a = dict(heads=4, kv=2, dim=8, mul=1 << 14, q=Fake((5, 4, 8)), k=Fake((5, 2, 8)), v=Fake((5, 2, 8)), cu=Fake((3,)), out=Fake((5, 4, 8), ptr=1 << 41), ws=Fake((1 << 22,), "uint8"))
    a.update(kw)
    at = T.Attention(a["heads"], a["kv"], a["dim"], a["mul"])
    at.prompt(a["q"], a["k"], a["v"], a["cu"], a["out"], a["ws"])


@pytest.mark.parametrize("kw,why", [
    (dict(heads=4, kv=3, k=Fake((5, 3, 8)), v=Fake((5, 3, 8))), "must divide"),
    (dict(heads=0, q=Fake((5, 0, 8)), out=Fake((5, 0, 8))), "must divide"),
    (dict(dim=257, q=Fake((5, 4, 257)), k=Fake((5, 2, 257)), v=Fake((5, 2, 257)), out=Fake((5, 4, 257))), "head_dim"),
    (dict(mul=0), "score_mul"), (dict(mul=(1 << 14) + 1), "score_mul"), (dict(mul=-5), "score_mul"),
    (dict(q=Fake((5, 4, 8), strides=(32, 4, 1))), "strides"),
    (dict(out=Fake((5, 4, 8), strides=(8, 8, 1))), "overlap"), (dict(out=Fake((5, 4, 8))), "may not be"),
    (dict(out=Fake((5, 4, 8), strides=(0, 8, 1))), "strides"),
    (dict(q=Fake((5, 4, 8), ptr=(1 << 40) + 2)), "aligned"),
    (dict(ws=Fake((8,), "uint8")), "workspace"),
    (dict(ws=Fake((1 << 22,), "uint8", ptr=(1 << 40) + 8)), "workspace"),
    (dict(cu=Fake((3,), ptr=0)), "cu_seqlens"),
    (dict(v=Fake((5, 2, 8), ptr=0)), "null"),
])
def test_prompt_refusals(kw, why):
    import jolt_atlas_amd as A
    with pytest.raises(A.AtlasError, match=why):
        _prompt(**kw)


@pytest.mark.parametrize("kw", [dict(q=Fake((5, 4, 8), "int64")), dict(k=Fake((4, 2, 8))), dict(out=Fake((6, 4, 8))), dict(cu=Fake((0,))), dict(cu=Fake((3,), strides=(2,))),
                                dict(q=Fake((5, 4, 8), strides=(64, 16, 2))), dict(v=Fake((5, 8)))])
def test_prompt_refusals_of_the_wrapper(kw):
    with pytest.raises(ValueError):
        _prompt(**kw)


def _cached(**kw):
    import jolt_atlas_amd.attention as T
    a = dict(q=Fake((3, 4, 8)), cu=Fake((3,)), lens=Fake((2,)), ck=Fake((7, 2, 16, 8)), cv=Fake((7, 2, 16, 8)), table=Fake((2, 5)), out=Fake((3, 4, 8), ptr=1 << 41), ws=Fake((1 << 22,), "uint8"))
    a.update(kw)
    T.Attention(4, 2, 8).cached(a["q"], a["cu"], a["lens"], T.KVCache(a["ck"], a["cv"]), a["table"], a["out"], a["ws"])


@pytest.mark.parametrize("kw,why", [
    (dict(ck=Fake((7, 2, 24, 8)), cv=Fake((7, 2, 24, 8))), "block_size"),
    (dict(ck=Fake((7, 2, 8192, 8)), cv=Fake((7, 2, 8192, 8))), "block_size"),
    (dict(ck=Fake((0, 2, 16, 8)), cv=Fake((0, 2, 16, 8))), "n_blocks"),
    (dict(ck=Fake((7, 2, 16, 8), ptr=(1 << 40) + 2)), "alignment"),
    (dict(cv=Fake((7, 2, 16, 8), ptr=0)), "null"),
    (dict(lens=Fake((2,), ptr=0)), "null"),
    (dict(out=Fake((3, 4, 8))), "may not be"),
    (dict(table=Fake((2, 1 << 28))), "table_stride"),
    (dict(ws=Fake((8,), "uint8")), "workspace"),
])
def test_cached_refusals(kw, why):
    import jolt_atlas_amd as A
    with pytest.raises(A.AtlasError, match=why):
        _cached(**kw)


@pytest.mark.parametrize("kw", [dict(ck=Fake((7, 2, 16, 8), "int16")), dict(ck=Fake((7, 2, 16, 8), "int64"), cv=Fake((7, 2, 16, 8), "int64")), dict(ck=Fake((7, 3, 16, 8)), cv=Fake((7, 3, 16, 8))),
                                dict(table=Fake((1, 5))), dict(lens=Fake((1,))), dict(ck=Fake((7, 2, 16, 8), strides=(256, 8, 16, 1)))])
def test_cached_refusals_of_the_wrapper(kw):
    with pytest.raises(ValueError):
        _cached(**kw)


def _plan(block=16, n_blocks=9, **kw):
    import jolt_atlas_amd.attention as T
    a = dict(have=Fake((2,)), new=Fake((2,)), table=Fake((2, 5)), free=Fake((9,)), n_free=Fake((1,)), n_out=Fake((1,)), cu=Fake((3,)), lens=Fake((2,), ptr=1 << 41), slots=Fake((6,), "int64"),
             pos=Fake((6,)), status=Fake((1,)), ws=Fake((1 << 12,), "uint8"))
    a.update(kw)
    T.Pager(block, n_blocks).plan(a["have"], a["new"], a["table"], a["free"], a["n_free"], a["n_out"], a["cu"], a["lens"], a["slots"], a["pos"], a["status"], a["ws"])


@pytest.mark.parametrize("kw,why", [
    (dict(block=12), "block_size"), (dict(block=0), "block_size"), (dict(n_blocks=0), "n_blocks"), (dict(lens=Fake((2,))), "may not be"), (dict(ws=Fake((16,), "uint8")), "workspace"),
    (dict(status=Fake((1,), ptr=0)), "null"), (dict(slots=Fake((6,), "int64", ptr=(1 << 40) + 4)), "aligned"), (dict(have=Fake((2,), ptr=0)), "null"),
])
def test_plan_refusals(kw, why):
    import jolt_atlas_amd as A
    with pytest.raises(A.AtlasError, match=why):
        _plan(**kw)


@pytest.mark.parametrize("kw", [dict(free=Fake((8,))), dict(table=Fake((1, 5))), dict(cu=Fake((2,))), dict(pos=Fake((5,))), dict(slots=Fake((6,))), dict(new=Fake((2,), "int64"))])
def test_plan_refusals_of_the_wrapper(kw):
    with pytest.raises(ValueError):
        _plan(**kw)


def test_write_refusals():
    import jolt_atlas_amd as A
    import jolt_atlas_amd.attention as T
    cache = T.KVCache(Fake((7, 2, 16, 8)), Fake((7, 2, 16, 8)))
    with pytest.raises(A.AtlasError, match="slots"):
        cache.write(Fake((5, 2, 8)), Fake((5, 2, 8)), Fake((5,), "int64", ptr=0))
    with pytest.raises(A.AtlasError, match="strides"):
        cache.write(Fake((5, 2, 8)), Fake((5, 2, 8), strides=(16, 4, 1)), Fake((5,), "int64"))
    for k, v, s in ((Fake((5, 2, 8)), Fake((4, 2, 8)), Fake((5,), "int64")), (Fake((5, 2, 8)), Fake((5, 2, 8)), Fake((4,), "int64")), (Fake((5, 2, 8)), Fake((5, 2, 8)), Fake((5,)))):
        with pytest.raises(ValueError):
            cache.write(k, v, s)


def test_workspace_sizes():
    import jolt_atlas_amd as A
    import jolt_atlas_amd.attention as T
    at = T.Attention(4, 2, 8)
    cache = T.KVCache(Fake((7, 2, 16, 8)), Fake((7, 2, 16, 8)))
    assert at.prompt_workspace_bytes(3, 100) > 0 and at.cached_workspace_bytes(3, 3, cache, 5) > 0
    for bad in (lambda: at.prompt_workspace_bytes(1 << 25, 4), lambda: at.prompt_workspace_bytes(1, (1 << 30) + 1), lambda: T.Attention(4, 3, 8).prompt_workspace_bytes(1, 1),
                lambda: at.cached_workspace_bytes(1, 1, cache, 1 << 28), lambda: T.Pager(16, 9).workspace_bytes(1 << 25, 4)):
        with pytest.raises(A.AtlasError):
            bad()
    assert A.lib.atlas_attn_prompt_workspace(C.POINTER(T._Shape)(), 1, 1) == 0


@pytest.mark.parametrize("n", [1 << 22, (1 << 22) + 5, 1 << 30])
def test_query_rows_past_32_bits_are_refused(n):
    """1024 heads over one kv head: the rows of a sequence are counted in 32 bits"""
    import jolt_atlas_amd as A
    import jolt_atlas_amd.attention as T
    ws, out = Fake((1 << 50,), "uint8"), Fake((n, 1024, 1), ptr=1 << 41)
    with pytest.raises(A.AtlasError, match="query rows"):
        _prompt(heads=1024, kv=1, dim=1, q=Fake((n, 1024, 1)), k=Fake((n, 1, 1)), v=Fake((n, 1, 1)), out=out, ws=ws)
    at, cache = T.Attention(1024, 1, 1, causal=False), T.KVCache(Fake((7, 1, 16, 1)), Fake((7, 1, 16, 1)))
    with pytest.raises(A.AtlasError, match="query rows"):
        at.cached(Fake((n, 1024, 1)), Fake((2,)), Fake((1,)), cache, Fake((1, 1)), out, ws)
    for f in (lambda: at.prompt_workspace_bytes(1, n), lambda: at.cached_workspace_bytes(1, n, cache, 1)):
        with pytest.raises(A.AtlasError):
            f()
    assert at.prompt_workspace_bytes(1, (1 << 22) - 1) > 0


@pytest.mark.parametrize("heads,kv,n,seqs,cols", [(64, 64, 1 << 17, 1 << 17, 4), (32, 32, 1 << 19, 1 << 19, 300), (32, 8, 1 << 19, 1 << 19, 300),
                                                  (32, 8, 100, 1 << 24, 300), (2, 1, 1 << 21, 1 << 14, 1 << 20)])
def test_more_than_a_launch_holds_is_refused(heads, kv, n, seqs, cols):
    """on the host, before the first of a path's launches"""
    import jolt_atlas_amd as A
    import jolt_atlas_amd.attention as T
    at, cache = T.Attention(heads, kv, 8), T.KVCache(Fake((7, kv, 16, 8)), Fake((7, kv, 16, 8)))
    with pytest.raises(A.AtlasError):
        at.cached_workspace_bytes(seqs, n, cache, cols)
    with pytest.raises(A.AtlasError, match="too many"):
        at.cached(Fake((n, heads, 8)), Fake((seqs + 1,)), Fake((seqs,)), cache, Fake((seqs, cols)), Fake((n, heads, 8), ptr=1 << 41), Fake((1 << 60,), "uint8"))


def test_more_tokens_than_a_launch_holds_are_refused():
    import jolt_atlas_amd as A
    import jolt_atlas_amd.attention as T
    at, n = T.Attention(1, 1, 8), 1 << 29
    with pytest.raises(A.AtlasError):
        at.prompt_workspace_bytes(1, n)
    with pytest.raises(A.AtlasError, match="too many"):
        at.prompt(*(Fake((n, 1, 8)) for _ in range(3)), Fake((2,)), Fake((n, 1, 8), ptr=1 << 41), Fake((1 << 60,), "uint8"))
    assert at.prompt_workspace_bytes(1, n - 1024) > 0
    # 2^17 tokens of 64 heads over one: 655360 workgroups of 512 threads, below 2^32 of them
    assert T.Attention(64, 1, 8).cached_workspace_bytes(1 << 17, 1 << 17, T.KVCache(Fake((7, 1, 16, 8)), Fake((7, 1, 16, 8))), 4) > 0


@pytest.mark.parametrize("status", [Fake((1,), "int8"), Fake((4,), "uint8"), Fake((1,), "bool"), Fake((1,), "int64"), Fake((0,)), Fake((3, 0))])
def test_a_status_that_is_no_32_bit_word(status):
    import jolt_atlas_amd.attention as T
    cache = T.KVCache(Fake((7, 2, 16, 8)), Fake((7, 2, 16, 8)))
    with pytest.raises(ValueError, match="status"):
        cache.write(Fake((5, 2, 8)), Fake((5, 2, 8)), Fake((5,), "int64"), status)
    with pytest.raises(ValueError, match="status"):
        _plan(status=status)


@pytest.mark.parametrize("off", [1, 2, 3])
def test_a_status_that_is_not_aligned(off):
    import jolt_atlas_amd as A
    import jolt_atlas_amd.attention as T
    cache, status = T.KVCache(Fake((7, 2, 16, 8)), Fake((7, 2, 16, 8))), Fake((1,), "uint32", ptr=(1 << 40) + off)
    with pytest.raises(A.AtlasError, match="status must be 4-byte"):
        cache.write(Fake((5, 2, 8)), Fake((5, 2, 8)), Fake((5,), "int64"), status)
    with pytest.raises(A.AtlasError, match="status must be 4-byte"):
        _plan(status=status)


@pytest.mark.parametrize("off", [1, 2, 3])
def test_offsets_tables_and_lengths_that_are_not_aligned(off):
    import jolt_atlas_amd as A
    at = (1 << 40) + off
    with pytest.raises(A.AtlasError, match="4-byte"):
        _prompt(cu=Fake((3,), ptr=at))
    for kw in (dict(cu=Fake((3,), ptr=at)), dict(lens=Fake((2,), ptr=at)), dict(table=Fake((2, 5), ptr=at))):
        with pytest.raises(A.AtlasError, match="4-byte"):
            _cached(**kw)
    for kw in (dict(have=Fake((2,), ptr=at)), dict(new=Fake((2,), ptr=at)), dict(table=Fake((2, 5), ptr=at)), dict(free=Fake((9,), ptr=at)), dict(n_free=Fake((1,), ptr=at)),
               dict(n_out=Fake((1,), ptr=at)), dict(cu=Fake((3,), ptr=at)), dict(lens=Fake((2,), ptr=(1 << 41) + off)), dict(pos=Fake((6,), ptr=at))):
        with pytest.raises(A.AtlasError, match="4-byte"):
            _plan(**kw)


@pytest.mark.parametrize("ws", [Fake((1 << 22,), "uint8", strides=(0,)), Fake((1 << 22,), "uint8", strides=(2,)), Fake((1 << 11, 1 << 11), "uint8", strides=(0, 1))])
def test_a_workspace_that_is_not_all_there(ws):
    """an expanded array is as long as its shape says and has the memory of one element"""
    for call in (_prompt, _cached, _plan):
        with pytest.raises(ValueError, match="workspace"):
            call(ws=ws)


@pytest.mark.parametrize("mul", [(1 << 32) + 2048, -(1 << 32) + 1, 1 << 31])
def test_a_score_mul_that_32_bits_do_not_hold(mul):
    with pytest.raises(ValueError, match="score_mul"):
        _prompt(mul=mul)


def test_steps_without_tokens_or_sequences():
    """empty arrays have no address (torch's is 0): nothing is enqueued and nothing is wrong"""
    import jolt_atlas_amd.attention as T
    none = lambda *shape, dtype="int32": Fake(shape, dtype, ptr=0)  # noqa: E731
    cache = T.KVCache(Fake((7, 2, 16, 8)), Fake((7, 2, 16, 8)))
    cache.write(none(0, 2, 8), none(0, 2, 8), none(0, dtype="int64"))
    at, ws = T.Attention(4, 2, 8), Fake((1 << 22,), "uint8")
    rows = none(0, 4, 8)
    assert at.cached(rows, Fake((1,)), none(0), cache, none(0, 5), rows, ws) is rows                  # no requests
    assert at.cached(rows, Fake((3,)), Fake((2,)), cache, Fake((2, 5)), rows, ws) is rows             # all of them pause
    assert at.cached(rows, Fake((3,)), Fake((2,)), cache, none(2, 0), rows, ws) is rows
    out = Fake((5, 4, 8), ptr=1 << 41)
    assert at.cached(Fake((5, 4, 8)), Fake((1,)), none(0), cache, none(0, 5), out, ws) is out         # only padding
    assert at.prompt(rows, none(0, 2, 8), none(0, 2, 8), Fake((1,)), rows, ws) is rows


def test_a_workspace_serves_smaller_calls():
    """the sizes do not decrease in any argument"""
    import jolt_atlas_amd.attention as T
    rng = np.random.default_rng(17)
    for _ in range(3000):
        kv, group, d, block = int(rng.choice([1, 2, 5, 8, 16, 64])), int(rng.choice([1, 2, 3, 8, 40])), int(rng.choice([1, 16, 64, 80, 128, 200, 256])), int(rng.choice([1, 16, 128]))
        if kv * group > 1024:
            continue
        at, cache = T.Attention(kv * group, kv, d), T.KVCache(*(Fake((7, kv, block, d)) for _ in range(2)))
        small = [int(np.exp(rng.uniform(0, np.log(x)))) for x in (300, 20000, 20000)]
        large = [x if rng.random() < 0.3 else x + int(np.exp(rng.uniform(0, np.log(x + 300)))) for x in small]
        size = lambda a: at.cached_workspace_bytes(a[0], a[1], cache, -(-a[2] // block))  # noqa: E731
        assert size(small) <= size(large), (kv, group, d, block, small, large)
        assert at.prompt_workspace_bytes(*small[:2]) <= at.prompt_workspace_bytes(*large[:2]), (kv, group, d, small, large)


@pytest.mark.parametrize("n", [0, 1, 2, 15, 16, 33, 64])
def test_a_serving_steps_workspace_serves_fewer_requests(n):
    """16 heads of 64, 125 blocks of 16: 16 single tokens are one launch, which needs nothing, fewer are not"""
    import jolt_atlas_amd as A
    import jolt_atlas_amd.attention as T
    at, cache = T.Attention(16, 16, 64), T.KVCache(*(Fake((7, 16, 16, 64)) for _ in range(2)))
    ws = Fake((at.cached_workspace_bytes(64, 64, cache, 125),), "uint8")
    try:
        at.cached(Fake((n, 16, 64)), Fake((n + 1,)), Fake((n,)), cache, Fake((n, 125)), Fake((n, 16, 64), ptr=1 << 41), ws)
    except A.AtlasError as e:               # no device here, or addresses that are not its
        assert "workspace" not in str(e)


@pytest.mark.parametrize("seqs,tokens", [(0, 0), (0, 1), (0, 900), (3, 0), (1, 1)])
def test_a_workspace_of_the_size_asked_for(seqs, tokens):
    import jolt_atlas_amd as A
    import jolt_atlas_amd.attention as T
    at, cache = T.Attention(16, 16, 64), T.KVCache(*(Fake((7, 16, 16, 64)) for _ in range(2)))
    for cols in (1, 125, 4000):
        q, out = Fake((tokens, 16, 64)), Fake((tokens, 16, 64), ptr=1 << 41)
        calls = [lambda: at.cached(q, Fake((seqs + 1,)), Fake((seqs,)), cache, Fake((seqs, cols)), out, Fake((at.cached_workspace_bytes(seqs, tokens, cache, cols),), "uint8")),
                 lambda: at.prompt(q, q, q, Fake((seqs + 1,)), out, Fake((at.prompt_workspace_bytes(seqs, tokens),), "uint8"))]
        for f in calls:
            try:
                f()
            except A.AtlasError as e:       # no device here, or addresses that are not its
                assert seqs and tokens and "workspace" not in str(e)


def test_the_stream_of_torch_tensors(monkeypatch):
    """without a stream of the caller's: torch's current one for torch tensors (0, its default, is the null stream), the library's for other arrays"""
    import sys
    import types
    import jolt_atlas_amd.attention as T

    class Tensor(Fake):
        is_cuda, device = True, "cuda:0"

    now = types.SimpleNamespace(cuda_stream=77)
    monkeypatch.setitem(sys.modules, "torch", types.SimpleNamespace(Tensor=Tensor, cuda=types.SimpleNamespace(current_stream=lambda dev: now if dev == "cuda:0" else None)))
    seen = {}
    for name in ("atlas_attn_prompt", "atlas_attn_cached", "atlas_kv_write", "atlas_kv_plan"):
        monkeypatch.setattr(T.lib, name, lambda *a, name=name: seen.__setitem__(name, a[-1]) or 0)

    def streams(kind, **kw):
        seen.clear()
        t = lambda shape, dtype="int32", ptr=1 << 40: kind(shape, dtype, ptr=ptr)  # noqa: E731
        at, cache, ws = T.Attention(4, 2, 8), T.KVCache(t((7, 2, 16, 8)), t((7, 2, 16, 8))), t((1 << 22,), "uint8")
        at.prompt(t((5, 4, 8)), t((5, 2, 8)), t((5, 2, 8)), t((3,)), t((5, 4, 8), ptr=1 << 41), ws, **kw)
        at.cached(t((3, 4, 8)), t((3,)), t((2,)), cache, t((2, 5)), t((3, 4, 8), ptr=1 << 41), ws, **kw)
        cache.write(t((5, 2, 8)), t((5, 2, 8)), t((5,), "int64"), **kw)
        T.Pager(16, 9).plan(t((2,)), t((2,)), t((2, 5)), t((9,)), t((1,)), t((1,)), t((3,)), t((2,)), t((6,), "int64"), None, t((1,)), ws, **kw)
        assert len(seen) == 4 and len(set(seen.values())) == 1
        return seen["atlas_kv_plan"]

    assert streams(Fake) is None and streams(Tensor) == 77
    now.cuda_stream = 0
    assert streams(Tensor) == 1 and streams(Tensor, stream=5) == 5 and streams(Tensor, stream=0) == 1 and streams(Fake, stream=9) == 9
    assert streams(Tensor, stream=T.LIBRARY_STREAM) is None and streams(Fake, stream=T.LIBRARY_STREAM) is None


def graph_attention(name):
    """the attention layers of one of the framework's graphs at its example input, run by the oracle's executor: q, k, v, the Mul constant, the Iff's fill, the output"""
    from tools import build_graphs
    from oracle import graph as OG
    nodes, _, inputs = getattr(build_graphs, name)()
    outs, _ = OG.execute(nodes, inputs)
    by = {nd["idx"]: nd for nd in nodes}
    for nd in nodes:
        if nd["op"] != "SoftmaxLastAxis":
            continue
        iff = by[nd["inputs"][0]]
        att, mul = by[iff["inputs"][1]], 1 << 14
        if att["op"] == "Mul":
            mul, att = int(outs[att["inputs"][1]].flat[0]), by[att["inputs"][0]]
        y = next(x for x in nodes if x["op"] == "Einsum" and x["inputs"][0] == nd["idx"])
        shape = (nd["dims"][1], nd["dims"][0], -1)
        yield tuple(np.ascontiguousarray(outs[i].reshape(shape)) for i in (*att["inputs"], y["inputs"][1])), mul, int(outs[iff["inputs"][2]].flat[0]), outs[y["idx"]].reshape(shape)


@pytest.mark.parametrize("name,fill,weighs", [("microgpt_model", -10, False), ("nanogpt_model", -10, False), ("nanogpt", -10, True), ("gpt2_layer", -8, True)])
def test_where_the_reference_is_the_frameworks_graphs(name, fill, weighs):
    """the framework's own graphs, whose mask fill is near: the same rows where no masked key weighs, and told where one does"""
    from _attention_ref import mask_weighs, prompt
    told = False
    for (q, k, v), mul, f, want in graph_attention(name):
        n = len(q)
        assert f == fill << 14
        got = prompt(q, k, v, [n], mul)
        for i in range(n):
            tell = mask_weighs(q[i:i + 1], k, [i + 1], [i], mul, f, n)
            assert tell or np.array_equal(got[i], want[i]), i
            told |= tell
    assert told == weighs


def _masked(mask=None, status=Fake((1,)), **kw):
    import jolt_atlas_amd.attention as T
    at, ws = T.Attention(4, 2, 8, mask_fill=-(10 << 14), mask_tokens=64, **kw), Fake((1 << 22,), "uint8")
    calls = [lambda: at.prompt(Fake((5, 4, 8)), Fake((5, 2, 8)), Fake((5, 2, 8)), Fake((3,)), Fake((5, 4, 8), ptr=1 << 41), ws, status=status),
             lambda: at.cached(Fake((3, 4, 8)), Fake((3,)), Fake((2,)), T.KVCache(*(Fake((7, 2, 16, 8)) for _ in range(2))), Fake((2, 5)), Fake((3, 4, 8), ptr=1 << 41), ws, status=status)]
    return calls


def test_mask_refusals():
    import jolt_atlas_amd as A
    import jolt_atlas_amd.attention as T
    for kw, why in ((dict(status=Fake((1,), ptr=0)), "status is null"), (dict(status=Fake((1,), ptr=(1 << 40) + 2)), "4-byte"), (dict(causal=False), "causal")):
        for f in _masked(**kw):
            with pytest.raises(A.AtlasError, match=why):
                f()
    for f in _masked(status=Fake((1,), "int64")) + _masked(status=Fake((0,))):
        with pytest.raises(ValueError, match="status"):
            f()
    for kw in (dict(mask_fill=-5), dict(mask_tokens=64), dict(mask_fill=1 << 31, mask_tokens=64), dict(mask_fill=0, mask_tokens=0), dict(mask_fill=0, mask_tokens=1 << 31)):
        with pytest.raises(ValueError, match="mask"):
            T.Attention(4, 2, 8, **kw)
    at = T.Attention(4, 2, 8)
    with pytest.raises(ValueError, match="mask_fill"):
        at.prompt(Fake((5, 4, 8)), Fake((5, 2, 8)), Fake((5, 2, 8)), Fake((3,)), Fake((5, 4, 8), ptr=1 << 41), Fake((1 << 22,), "uint8"), status=Fake((1,)))
    null, rows, cache = C.POINTER(T._Mask)(), T._Rows(1 << 40, 32, 8), T.KVCache(*(Fake((7, 2, 16, 8)) for _ in range(2)))
    assert A.lib.atlas_attn_prompt_masked(C.byref(at.shape), *[C.byref(rows)] * 3, 1 << 40, 1, 1, C.byref(T._Rows(1 << 41, 32, 8)), null, 1 << 40, 1 << 22, None) != 0
    assert A.lib.atlas_attn_cached_masked(C.byref(at.shape), C.byref(rows), 1 << 40, 1 << 40, 1, 1, C.byref(cache.desc), 1 << 40, 1, 1, C.byref(T._Rows(1 << 41, 32, 8)), null,
                                          1 << 40, 1 << 22, None) != 0
    assert "mask" in A.lib.atlas_last_error().decode()
    for n in (0, 1 << 31):
        m = T._Mask(0, n, 1 << 40)
        assert A.lib.atlas_attn_prompt_masked(C.byref(at.shape), *[C.byref(rows)] * 3, 1 << 40, 1, 1, C.byref(T._Rows(1 << 41, 32, 8)), C.byref(m), 1 << 40, 1 << 22, None) != 0
        assert "n_tokens" in A.lib.atlas_last_error().decode()
