"""Quantised attention for generation (atlas_attn_*, atlas_kv_*): ctypes marshalling only.

The attention of a model graph in the graph executor's integers — over packed prompts (Attention.prompt) and over a paged cache of keys and
values (Attention.cached) —, the cache and its write (KVCache), and the paging of a step from request lengths (Pager).  A row in which the graph's masked keys
carry no weight comes out bit for bit as graph.Graph.trace has it, so that what was generated is what atlas_prove_graph proves; whether they carry none goes by the
graph's mask fill and the inputs, and a call's `status` tells.

Tensors are device arrays of anything that has data_ptr(), shape, stride() and dtype (torch tensors do); they are used in place, on the calling thread's
device (init / init_thread).  A process that uses torch imports it before this package: the one HIP runtime is then torch's.

stream: a hipStream_t as an integer (torch: torch.cuda.current_stream().cuda_stream, whose 0 is HIP's default stream), or LIBRARY_STREAM, the stream that the library's
other calls run on and that no other stream waits for or is waited for by.  None: torch's current stream where the arrays are torch tensors, so that a call comes after what
made its inputs; the library stream for other arrays.  Calls enqueue and return; nothing is kept between them, so a call may be captured into a graph."""
import ctypes as C
import sys

from . import AtlasError, _check, lib

ONE = 1 << 14                       # scale 2^14; the score_mul that scales nothing
LIBRARY_STREAM = "library"          # stream=
NARROW, BAD_SLOT = 1, 2             # KVCache.write's status
MASK_WEIGHS = 1                     # Attention.prompt's and .cached's status
NO_BLOCKS, NO_COLUMNS, NO_TOKENS, BAD_LENGTH = 1, 2, 4, 8      # Pager.plan's status


class _Shape(C.Structure):
    _fields_ = [("n_heads", C.c_size_t), ("n_kv_heads", C.c_size_t), ("head_dim", C.c_size_t), ("score_mul", C.c_int32), ("causal", C.c_int32)]


class _Rows(C.Structure):
    _fields_ = [("d", C.c_void_p), ("token_stride", C.c_size_t), ("head_stride", C.c_size_t)]


class _Cache(C.Structure):
    _fields_ = [("d_k", C.c_void_p), ("d_v", C.c_void_p), ("n_blocks", C.c_size_t), ("block_size", C.c_size_t), ("bits", C.c_int32)]


class _Mask(C.Structure):
    _fields_ = [("fill", C.c_int32), ("n_tokens", C.c_uint32), ("d_status", C.c_void_p)]


_vp, _sz, _R, _S, _K, _M = C.c_void_p, C.c_size_t, C.POINTER(_Rows), C.POINTER(_Shape), C.POINTER(_Cache), C.POINTER(_Mask)
lib.atlas_attn_prompt_workspace.argtypes, lib.atlas_attn_prompt_workspace.restype = [_S, _sz, _sz], _sz
lib.atlas_attn_prompt.argtypes, lib.atlas_attn_prompt.restype = [_S, _R, _R, _R, _vp, _sz, _sz, _R, _vp, _sz, _vp], C.c_int
lib.atlas_attn_cached_workspace.argtypes, lib.atlas_attn_cached_workspace.restype = [_S, _sz, _sz, _K, _sz], _sz
lib.atlas_attn_cached.argtypes, lib.atlas_attn_cached.restype = [_S, _R, _vp, _vp, _sz, _sz, _K, _vp, _sz, _sz, _R, _vp, _sz, _vp], C.c_int
lib.atlas_attn_prompt_masked.argtypes, lib.atlas_attn_prompt_masked.restype = [_S, _R, _R, _R, _vp, _sz, _sz, _R, _M, _vp, _sz, _vp], C.c_int
lib.atlas_attn_cached_masked.argtypes, lib.atlas_attn_cached_masked.restype = [_S, _R, _vp, _vp, _sz, _sz, _K, _vp, _sz, _sz, _R, _M, _vp, _sz, _vp], C.c_int
lib.atlas_kv_write.argtypes, lib.atlas_kv_write.restype = [_S, _R, _R, _vp, _sz, _K, _vp, _vp], C.c_int
lib.atlas_kv_plan_workspace.argtypes, lib.atlas_kv_plan_workspace.restype = [_sz, _sz], _sz
lib.atlas_kv_plan.argtypes, lib.atlas_kv_plan.restype = [_sz, _sz, _vp, _vp, _sz, _vp, _sz, _sz, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _sz, _vp, _vp, _sz, _vp], C.c_int


def _stream(stream, t):
    """the entry points' stream argument; t: one of the call's arrays"""
    if stream is None:
        torch = sys.modules.get("torch")
        if torch is None or not isinstance(t, torch.Tensor) or not t.is_cuda:
            return None
        stream = torch.cuda.current_stream(t.device).cuda_stream
    return None if stream is LIBRARY_STREAM else (stream or 1)          # ATLAS_STREAM_DEFAULT


_names = {}                         # dtype -> "int32", ...: a call looks its arrays' types up six times


def _name(dtype):
    n = _names.get(dtype)
    if n is None:
        n = _names[dtype] = str(dtype).rpartition(".")[2]
    return n


def _is(t, name, dtype, ndim):
    if len(t.shape) != ndim or _name(t.dtype) != dtype:
        raise ValueError(f"{name}: a {ndim}-dimensional {dtype} array expected, got {t.dtype} {tuple(t.shape)}")


def _vector(t, name, dtype, n=None):
    """a contiguous array of `n` elements (None: any number), as a pointer"""
    shape = t.shape
    if len(shape) != 1 or _name(t.dtype) != dtype:
        _is(t, name, dtype, 1)
    if n is not None and shape[0] < n:
        raise ValueError(f"{name}: {n} elements expected, got {shape[0]}")
    if shape[0] > 1 and t.stride()[0] != 1:
        raise ValueError(f"{name}: a contiguous array expected")
    return t.data_ptr()


def _rows(t, name, heads, dim):
    shape = t.shape
    if len(shape) != 3 or _name(t.dtype) != "int32":
        _is(t, name, "int32", 3)
    n, h, d = shape
    if h != heads or d != dim:
        raise ValueError(f"{name}: [tokens][{heads}][{dim}] expected, got {tuple(shape)}")
    if n == 0:
        return _Rows(t.data_ptr(), heads * dim, dim)
    a, b, c = t.stride()
    if c != 1 and dim > 1 or a < 0 or b < 0:
        raise ValueError(f"{name}: the elements of a head must be contiguous")
    return _Rows(t.data_ptr(), a if n > 1 else max(a, dim), b if heads > 1 else max(b, dim))


def _table(t):
    _is(t, "block_table", "int32", 2)
    if t.shape[1] > 1 and t.stride()[1] != 1:
        raise ValueError("block_table: the entries of a row must be contiguous")
    return t.data_ptr(), t.shape[1], max(t.stride()[0], t.shape[1])


def _status(t):
    """one 32-bit word that the kernels write: any array of at least one element"""
    if _name(t.dtype) not in ("int32", "uint32") or 0 in t.shape:
        raise ValueError(f"status: one int32 or uint32 expected, got {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


def _contiguous(t, name):
    want = 1
    for n, s in zip(reversed(t.shape), reversed(t.stride())):
        if n > 1 and s != want:
            raise ValueError(f"{name}: a contiguous array expected")
        want *= n
    return want


def _workspace(w):
    shape = w.shape
    n = shape[0] if len(shape) == 1 and w.stride()[0] == 1 else _contiguous(w, "workspace")
    return w.data_ptr(), n * w.itemsize


class KVCache:
    """one layer's paged cache over two arrays [n_blocks][n_kv_heads][block_size][head_dim] of the caller's, int32 or int16"""

    def __init__(self, k, v):
        if len(k.shape) != 4 or tuple(k.shape) != tuple(v.shape) or str(k.dtype) != str(v.dtype):
            raise ValueError("KVCache: two arrays [n_blocks][n_kv_heads][block_size][head_dim] of one type expected")
        bits = {"int32": 32, "int16": 16}.get(_name(k.dtype))
        if bits is None:
            raise ValueError(f"KVCache: int32 or int16 expected, got {k.dtype}")
        _contiguous(k, "KVCache: k"), _contiguous(v, "KVCache: v")
        self.k, self.v = k, v
        self.n_blocks, self.n_kv_heads, self.block_size, self.head_dim = k.shape
        self.desc = _Cache(k.data_ptr(), v.data_ptr(), self.n_blocks, self.block_size, bits)
        self._shape = _Shape(self.n_kv_heads, self.n_kv_heads, self.head_dim, ONE, 1)

    def write(self, k, v, slots, status=None, stream=None):
        """rows [tokens][n_kv_heads][head_dim] of k and v into `slots` (int64 [tokens]; negative: skipped).  status: one uint32 / int32 on the
        device that gets NARROW / BAD_SLOT ored in"""
        n = k.shape[0]
        if v.shape[0] != n:
            raise ValueError("KVCache.write: k and v have the same number of rows")
        _check(lib.atlas_kv_write(C.byref(self._shape), C.byref(_rows(k, "k", self.n_kv_heads, self.head_dim)), C.byref(_rows(v, "v", self.n_kv_heads, self.head_dim)),
                                  _vector(slots, "slots", "int64", n), n, C.byref(self.desc), None if status is None else _status(status), _stream(stream, k)))


class Attention:
    """score_mul: the Mul node's constant at scale 2^14 (round(2^14 / sqrt(head_dim)) is the usual; ONE: the graph has no such node).
    mask_fill, mask_tokens: what the graph's Iff fills masked scores with, and the graph's tokens; a call with a `status` then tells whether masked keys
    would weigh in the graph"""

    def __init__(self, n_heads, n_kv_heads, head_dim, score_mul=ONE, causal=True, mask_fill=None, mask_tokens=None):
        if not -(1 << 31) <= score_mul < 1 << 31:              # ctypes would cut it to 32 bits
            raise ValueError(f"Attention: score_mul must be 1 .. 2^14, got {score_mul}")
        self.n_heads, self.n_kv_heads, self.head_dim = n_heads, n_kv_heads, head_dim
        self.shape = _Shape(n_heads, n_kv_heads, head_dim, score_mul, 1 if causal else 0)
        if (mask_fill is None) != (mask_tokens is None):
            raise ValueError("Attention: mask_fill and mask_tokens belong together")
        if mask_fill is not None and not (-(1 << 31) <= mask_fill < 1 << 31 and 1 <= mask_tokens < 1 << 31):
            raise ValueError(f"Attention: mask_fill must fit 32 bits, mask_tokens must be 1 .. 2^31 - 1, got {mask_fill}, {mask_tokens}")
        self.mask_fill, self.mask_tokens = mask_fill, mask_tokens

    def prompt_workspace_bytes(self, n_seqs, n_tokens):
        return self._size(lib.atlas_attn_prompt_workspace(C.byref(self.shape), n_seqs, n_tokens))

    def cached_workspace_bytes(self, n_seqs, n_tokens, cache, max_blocks):
        return self._size(lib.atlas_attn_cached_workspace(C.byref(self.shape), n_seqs, n_tokens, C.byref(cache.desc), max_blocks))

    @staticmethod
    def _size(n):
        if n == 0:
            raise AtlasError("attention: the shape, the cache or the sizes are not supported")
        return n

    def _mask(self, status):
        if self.mask_fill is None:
            raise ValueError("Attention: a status needs mask_fill and mask_tokens")
        return C.byref(_Mask(self.mask_fill, self.mask_tokens, _status(status)))

    def prompt(self, q, k, v, cu_seqlens, out, workspace, stream=None, status=None):
        """q, out [tokens][n_heads][head_dim], k, v [tokens][n_kv_heads][head_dim], cu_seqlens int32 [n_seqs + 1]; returns out.  status: one uint32 / int32 on
        the device that gets MASK_WEIGHS ored in when the graph's masked keys would weigh in some row, so that its trace may be another"""
        n, n_seqs = q.shape[0], cu_seqlens.shape[0] - 1
        if n_seqs < 0 or not (k.shape[0] == v.shape[0] == out.shape[0] == n):
            raise ValueError("Attention.prompt: q, k, v and out have the same number of rows, cu_seqlens one entry more than sequences")
        p, size = _workspace(workspace)
        call, mask = (lib.atlas_attn_prompt, ()) if status is None else (lib.atlas_attn_prompt_masked, (self._mask(status),))
        _check(call(C.byref(self.shape), C.byref(_rows(q, "q", self.n_heads, self.head_dim)), C.byref(_rows(k, "k", self.n_kv_heads, self.head_dim)),
                    C.byref(_rows(v, "v", self.n_kv_heads, self.head_dim)), _vector(cu_seqlens, "cu_seqlens", "int32"), n_seqs, n,
                    C.byref(_rows(out, "out", self.n_heads, self.head_dim)), *mask, p, size, _stream(stream, q)))
        return out

    def cached(self, q, cu_new, kv_lens, cache, block_table, out, workspace, stream=None, status=None):
        """q, out [new tokens][n_heads][head_dim], cu_new int32 [n_seqs + 1], kv_lens int32 [n_seqs], block_table int32 [n_seqs][columns]; returns out.
        status: as for prompt"""
        n, n_seqs = q.shape[0], cu_new.shape[0] - 1
        if (cache.n_kv_heads, cache.head_dim) != (self.n_kv_heads, self.head_dim):
            raise ValueError("Attention.cached: the cache has other heads")
        if n_seqs < 0 or out.shape[0] != n or block_table.shape[0] < n_seqs:
            raise ValueError("Attention.cached: q and out have the same number of rows, cu_new one entry more than sequences, the table a row for each")
        p, size = _workspace(workspace)
        table, cols, stride = _table(block_table)
        call, mask = (lib.atlas_attn_cached, ()) if status is None else (lib.atlas_attn_cached_masked, (self._mask(status),))
        _check(call(C.byref(self.shape), C.byref(_rows(q, "q", self.n_heads, self.head_dim)), _vector(cu_new, "cu_new", "int32"),
                    _vector(kv_lens, "kv_lens", "int32", n_seqs), n_seqs, n, C.byref(cache.desc), table, cols, stride,
                    C.byref(_rows(out, "out", self.n_heads, self.head_dim)), *mask, p, size, _stream(stream, q)))
        return out


class Pager:
    """the paging of a step: which blocks the new tokens of each request go to (include/atlas_hip.h: atlas_kv_plan)"""

    def __init__(self, block_size, n_blocks):
        self.block_size, self.n_blocks = block_size, n_blocks

    def workspace_bytes(self, n_seqs, max_tokens):
        return Attention._size(lib.atlas_kv_plan_workspace(n_seqs, max_tokens))

    def plan(self, cached_lens, new_lens, block_table, free_blocks, n_free, n_free_out, cu_new, kv_lens, slots, positions, status, workspace, stream=None):
        """int32 arrays (slots: int64); positions may be None; len(slots) is the most new tokens a step may have"""
        n, cap = cached_lens.shape[0], slots.shape[0]
        p, size = _workspace(workspace)
        table, cols, stride = _table(block_table)
        if block_table.shape[0] < n:
            raise ValueError("Pager.plan: the table needs a row for each request")
        _check(lib.atlas_kv_plan(self.block_size, self.n_blocks, _vector(cached_lens, "cached_lens", "int32"), _vector(new_lens, "new_lens", "int32", n), n, table, cols, stride,
                                 _vector(free_blocks, "free_blocks", "int32", self.n_blocks), _vector(n_free, "n_free", "int32", 1), _vector(n_free_out, "n_free_out", "int32", 1),
                                 _vector(cu_new, "cu_new", "int32", n + 1), _vector(kv_lens, "kv_lens", "int32", n), _vector(slots, "slots", "int64"),
                                 None if positions is None else _vector(positions, "positions", "int32", cap), cap, _status(status), p, size, _stream(stream, cached_lens)))
