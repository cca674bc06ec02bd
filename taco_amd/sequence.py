"""The sequence memory of a policy on libtaco_sequence.so (include/taco_sequence.h): attention over whole episodes and over a paged cache, and linear
attention with a decay for each head, each in the form that training needs (packed sequences, with gradients) and the one that acting needs (one token per
row and call).  The reference's policies remember through frame stacks and an LSTM over them (nets_asymmetry.py:128-136); these hold any length.

    seqs = sequence.Packed(lengths, "cuda:0")             # once per rollout; RolloutBuffer.episodes() makes one from the done flags
    out = sequence.attention(q, k, v, seqs)               # q [T, heads, dim], k and v [T, kv_heads, dim]; causal inside each sequence; autograd
    out = sequence.attention_step(q, k, v, k_pages, v_pages, page_table, lengths)        # q [rows, heads, dim]: the token joins the cache
    lengths += 1                                          # (and lengths.masked_fill_(env.reset_buf.bool(), 0) where an episode ended)

    out, state = sequence.linear_attention(q, k, v, log_decay, seqs, state=state0)
    out = sequence.linear_attention_step(q, k, v, log_decay, state, reset=env.reset_buf)

float32, float16 and bfloat16; head dimensions that are multiples of 8 up to 128; sums, softmax statistics and states are float32.  Work is enqueued on the
current stream of the tensors' device, nothing synchronises, and every call gives the same bits each time.  There is no torch fallback.

HIP graphs: call once eagerly before capturing (the work lists are uploaded at the first call with a given number of heads), keep the Packed alive as long as
the graph, and capture a backward pass only while no eager autograd graph of the same leaf tensors is alive: torch then waits for the eager graph's stream
inside the capture, which it does not survive.
"""
import ctypes as C
import math

import numpy as np
import torch

from . import _lib

ABI_VERSION = 1
EXPORTS = ["taco_sequence_abi_version", "taco_sequence_source_hash", "taco_sequence_last_error", "taco_attention", "taco_attention_backward",
           "taco_attention_step_workspace_bytes", "taco_attention_step", "taco_linear_attention_workspace_bytes", "taco_linear_attention",
           "taco_linear_attention_backward", "taco_linear_attention_step"]
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


class Tensor(C.Structure):
    """struct taco_seq_tensor"""
    _fields_ = [("ptr", C.c_void_p), ("token_stride", C.c_int64), ("head_stride", C.c_int64)]


class AttentionArgs(C.Structure):
    """struct taco_attention_args"""
    _fields_ = [("q", Tensor), ("k", Tensor), ("v", Tensor), ("o", Tensor), ("lse", C.c_void_p), ("tiles", C.c_void_p), ("key_tiles", C.c_void_p),
                ("n_tiles", C.c_int32), ("tile_rows", C.c_int32), ("heads", C.c_int32), ("kv_heads", C.c_int32), ("dim", C.c_int32), ("dtype", C.c_int32),
                ("causal", C.c_int32), ("scale", C.c_float), ("d_o", Tensor), ("d_q", Tensor), ("d_k", Tensor), ("d_v", Tensor), ("delta", C.c_void_p)]


class AttentionStepArgs(C.Structure):
    """struct taco_attention_step_args"""
    _fields_ = [("q", Tensor), ("o", Tensor), ("k_new", Tensor), ("v_new", Tensor), ("k_pages", C.c_void_p), ("v_pages", C.c_void_p),
                ("k_page_stride", C.c_int64), ("k_token_stride", C.c_int64), ("k_head_stride", C.c_int64),
                ("v_page_stride", C.c_int64), ("v_token_stride", C.c_int64), ("v_head_stride", C.c_int64),
                ("table", C.c_void_p), ("table_stride", C.c_int64), ("lengths", C.c_void_p), ("rows", C.c_int32), ("table_width", C.c_int32),
                ("num_pages", C.c_int32), ("page_size", C.c_int32), ("heads", C.c_int32), ("kv_heads", C.c_int32), ("dim", C.c_int32), ("dtype", C.c_int32),
                ("scale", C.c_float), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


class LinearArgs(C.Structure):
    """struct taco_linear_attention_args"""
    _fields_ = [("q", Tensor), ("k", Tensor), ("v", Tensor), ("o", Tensor), ("log_decay", C.c_void_p), ("state0", C.c_void_p), ("state_last", C.c_void_p),
                ("segments", C.c_void_p), ("first_segment", C.c_void_p), ("n_segments", C.c_int32), ("n_sequences", C.c_int32),
                ("heads", C.c_int32), ("dim", C.c_int32), ("dtype", C.c_int32), ("scale", C.c_float), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
                ("d_o", Tensor), ("d_q", Tensor), ("d_k", Tensor), ("d_v", Tensor), ("d_state_last", C.c_void_p), ("d_state0", C.c_void_p)]


class LinearStepArgs(C.Structure):
    """struct taco_linear_attention_step_args"""
    _fields_ = [("q", Tensor), ("k", Tensor), ("v", Tensor), ("o", Tensor), ("log_decay", C.c_void_p), ("state", C.c_void_p), ("reset", C.c_void_p),
                ("reset_bytes", C.c_int32), ("rows", C.c_int32), ("heads", C.c_int32), ("dim", C.c_int32), ("dtype", C.c_int32), ("scale", C.c_float)]


_loaded = None


def load():
    """dlopen libtaco_sequence.so (built first if it is missing or stale) and declare its prototypes"""
    global _loaded
    if _loaded is None:
        import os
        from . import build
        if all(os.path.exists(os.path.join(build.CSRC, d)) for d in build.SEQ_DEPS):
            try:
                build.build_sequence()
            except Exception as e:  # noqa: BLE001 -- never a stale binary, never anything else in its place
                raise _lib.TacoError(f"{build.LIB_SEQ} is missing or stale and building it failed ({e}); run `python -m taco_amd.build` (hipcc, gfx950)") from e
        elif not os.path.exists(build.LIB_SEQ):
            raise _lib.TacoError(f"{build.LIB_SEQ} is missing and its sources are not next to the package")
        lib = C.CDLL(build.LIB_SEQ)
        lib.taco_sequence_source_hash.restype = lib.taco_sequence_last_error.restype = C.c_char_p
        for name, args in (("taco_attention", AttentionArgs), ("taco_attention_backward", AttentionArgs), ("taco_attention_step", AttentionStepArgs),
                           ("taco_linear_attention", LinearArgs), ("taco_linear_attention_backward", LinearArgs), ("taco_linear_attention_step", LinearStepArgs)):
            f = getattr(lib, name)
            f.argtypes, f.restype = [C.POINTER(args), C.c_void_p], C.c_int
        lib.taco_attention_step_workspace_bytes.argtypes, lib.taco_attention_step_workspace_bytes.restype = [C.POINTER(AttentionStepArgs)], C.c_size_t
        lib.taco_linear_attention_workspace_bytes.argtypes, lib.taco_linear_attention_workspace_bytes.restype = [C.POINTER(LinearArgs), C.c_int], C.c_size_t
        if lib.taco_sequence_abi_version() != ABI_VERSION:
            raise _lib.TacoError(f"libtaco_sequence.so ABI {lib.taco_sequence_abi_version()} != binding ABI {ABI_VERSION}")
        _loaded = lib
    return _loaded


def _call(name, args, device):
    lib = load()
    f = getattr(lib, name)
    if torch.cuda.current_device() == device.index:
        rc = f(C.byref(args), _lib.stream_ptr(device))
    else:                                       # a launch goes to the current device: make it the tensors'
        with torch.cuda.device(device):
            rc = f(C.byref(args), _lib.stream_ptr(device))
    if rc != 0:
        raise _lib.TacoError(f"libtaco_sequence: status {rc}: {lib.taco_sequence_last_error().decode()}")


# ---- checks shared by the calls ----------------------------------------------------------------------------------------------------

def _need(ok, message):
    if not ok:
        raise ValueError(message)


def _check_rows(named, what):
    """[rows, heads, dim] tensors of one supported dtype on one HIP device -> (device, dtype code)"""
    (n0, t0), device = named[0], named[0][1].device
    if device.type != "cuda":
        raise _lib.TacoError(f"{what} runs on an MI355X: {n0} has to be on a cuda:N (HIP) device")
    if t0.dtype not in _DTYPES:
        raise _lib.TacoError(f"{what}: {t0.dtype} is not supported (float32, float16, bfloat16)")
    for name, t in named:
        _need(t.dim() == 3, f"{name} of shape {tuple(t.shape)}: [tokens, heads, dim] expected")
        _need(t.device == device and t.dtype == t0.dtype, f"{name} is {t.dtype} on {t.device}, {n0} is {t0.dtype} on {device}")
        _need(t.shape[2] == t0.shape[2], f"{name} has head dimension {t.shape[2]}, {n0} has {t0.shape[2]}")
    d = t0.shape[2]
    if d % 8 or not 8 <= d <= 128:
        raise _lib.TacoError(f"{what}: head dimension {d} is not supported (a multiple of 8 from 8 to 128)")
    return device, _DTYPES[t0.dtype]


def _usable(t):
    """`t` itself if the kernels can address it (rows of whole 16-byte chunks that do not overlap), else a contiguous copy"""
    size = t.element_size()
    ok = t.stride(2) == 1 and t.data_ptr() % 16 == 0 and (t.shape[1] == 1 or (t.stride(1) * size) % 16 == 0 and t.stride(1) >= t.shape[2]) and \
        (t.shape[0] == 1 or (t.stride(0) * size) % 16 == 0 and t.shape[2] <= t.stride(0) <= 1 << 21)
    return t if ok else t.contiguous()


def _tensor(t):
    """of a tensor that _usable() returned; the stride of a dimension of one is never used"""
    d = t.shape[2]
    return Tensor(t.data_ptr(), t.stride(0) if t.shape[0] > 1 else t.shape[1] * d, t.stride(1) if t.shape[1] > 1 else d)


def _scale(scale, dim):
    return 1.0 / math.sqrt(dim) if scale is None else float(scale)


def _no_grad(tensors, what):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise _lib.TacoError(f"{what} has no gradient: call it under torch.no_grad(), or use the form over whole sequences")


class Packed:
    """Sequences behind one another in a tensor's first dimension: sequence i is rows [starts[i], starts[i] + lengths[i]).  `lengths`: non-negative whole numbers
    on the host (a list, an array, a CPU tensor); a device tensor is copied, which blocks.  Rows behind the last sequence may exist; no call reads them.
    Keeps the work lists of the kernels on `device`, made at the first call that needs them."""

    def __init__(self, lengths, device):
        n = lengths.detach().cpu().numpy() if isinstance(lengths, torch.Tensor) else np.asarray(lengths)
        _need(n.ndim == 1 and (n.size == 0 or np.issubdtype(n.dtype, np.integer)), "lengths: one whole number per sequence expected")
        n = n.astype(np.int64)
        _need(not (n < 0).any(), "lengths: a sequence cannot have a negative length")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise _lib.TacoError("the sequence kernels run on an MI355X; device must be a cuda:N (HIP) device")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.lengths, self.starts, self.total = n, np.cumsum(n) - n, int(n.sum())
        _need(self.total < 2 ** 31 - 4096, f"{self.total} tokens: fewer than 2^31 - 4096 are supported")
        self._lists = {}

    def __len__(self):
        return len(self.lengths)

    def _kept(self, key, make):
        """work list `key` on the device"""
        got = self._lists.get(key)
        if got is None:
            if torch.cuda.is_current_stream_capturing():
                raise _lib.TacoError("the work list of these sequences is not on the device yet: make one call before capturing a graph")
            got = self._lists[key] = [t if not isinstance(t, np.ndarray) else torch.from_numpy(np.ascontiguousarray(t)).to(self.device) for t in make()]
            self._lists[key].append(torch.cuda.current_stream(self.device).cuda_stream)
        elif got[-1] != (_lib.stream_ptr(self.device).value or 0) and not torch.cuda.is_current_stream_capturing():
            for t in got[:-1]:                  # a stream of its own: the memory is not given away before its work is done
                if isinstance(t, torch.Tensor):
                    t.record_stream(torch.cuda.current_stream(self.device))
        return got

    def _tiles(self, heads):
        """[(tile rows, tiles, key tiles, count)]: launches of 32- and of 128-row tiles.  A tile of 128 rows shares its loads between four wavefronts; sequences
        of at most 64 tokens would leave half of it idle, and where all tiles together do not fill the CUs, smaller ones spread the work."""
        big = self.lengths > 64
        if big.any() and (-(-self.lengths[big] // 128)).sum() * heads < 256:
            big = np.zeros_like(big)
        key = ("tiles", bool(big.any()))

        def make():
            out = []
            for rows, which in ((128, np.flatnonzero(big)), (32, np.flatnonzero(~big & (self.lengths > 0)))):
                n = -(-self.lengths[which] // rows)
                of = np.repeat(which, n)
                first = (np.arange(len(of)) - np.repeat(np.cumsum(n) - n, n)) * rows
                if len(of):
                    t = np.stack([self.starts[of], self.lengths[of], first, np.zeros_like(first)], 1).astype(np.int32)
                    out += [rows, t[np.argsort(-np.minimum(first + rows, self.lengths[of]), kind="stable")], t[np.argsort(first - self.lengths[of], kind="stable")], len(of)]
            return out
        got = self._kept(key, make)[:-1]
        return [got[i:i + 4] for i in range(0, len(got), 4)]

    def _segments(self, work):
        """(segments, first segment of each sequence, count) for `work` = heads x products: about 1 024 workgroups in all, segments of at least 256 tokens"""
        size = max(256, -(-self.total * work // (1024 * 64)) * 64)
        key = ("segments", size)

        def make():
            n = np.maximum(-(-self.lengths // size), 1)
            if len(n) and n.sum() > len(n) and len(n) * 128 > 65535:       # (the joining launch's limit; so many sequences fill the CUs by themselves)
                n = np.ones_like(n)
            first = np.concatenate([[0], np.cumsum(n)])
            of = np.repeat(np.arange(len(n)), n)
            index = np.arange(len(of)) - first[of]
            step = np.where(n[of] > 1, size, self.lengths[of])
            at = index * step
            cols = [of, self.starts[of], self.lengths[of], at, np.minimum(step, self.lengths[of] - at), index, index * 0, index * 0]
            return [np.stack(cols, 1).astype(np.int32).reshape(-1, 8), first.astype(np.int32), len(of)]
        return self._kept(key, make)[:3]


# ---- attention over packed sequences -----------------------------------------------------------------------------------------------

def _attention_args(q, k, v, o, lse, seqs, causal, scale):
    a = AttentionArgs()
    a.q, a.k, a.v, a.o = _tensor(q), _tensor(k), _tensor(v), _tensor(o)
    a.lse = lse.data_ptr()
    a.heads, a.kv_heads, a.dim, a.dtype = q.shape[1], k.shape[1], q.shape[2], _DTYPES[q.dtype]
    a.causal, a.scale = 1 if causal else 0, scale
    return a


def _launch_tiles(name, a, seqs, device):
    for rows, tiles, key_tiles, count in seqs._tiles(a.heads):
        a.tile_rows, a.tiles, a.key_tiles, a.n_tiles = rows, tiles.data_ptr(), key_tiles.data_ptr(), count
        _call(name, a, device)


def _empty(like, rows, total, dtype=None, shape=None):
    """uninitialised [rows, ...]; rows behind the last sequence are zero"""
    t = torch.empty((rows,) + tuple(like.shape[1:] if shape is None else shape), dtype=dtype or like.dtype, device=like.device)
    if rows > total:
        t[total:].zero_()
    return t


def _attention_forward(q, k, v, seqs, causal, scale, out):
    q, k, v = _usable(q), _usable(k), _usable(v)
    o = _empty(q, q.shape[0], seqs.total) if out is None else out
    lse = _empty(q, q.shape[0], seqs.total, torch.float32, (q.shape[1],))
    if seqs.total:
        _launch_tiles("taco_attention", _attention_args(q, k, v, o, lse, seqs, causal, scale), seqs, q.device)
    return q, k, v, o, lse


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, seqs, causal, scale):
        q, k, v, o, lse = _attention_forward(q, k, v, seqs, causal, scale, None)
        ctx.save_for_backward(q, k, v, o, lse)
        ctx.rest = seqs, causal, scale
        ctx.mark_non_differentiable(lse)
        return o, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_o, _):
        q, k, v, o, lse = ctx.saved_tensors
        seqs, causal, scale = ctx.rest
        d_o = _usable(d_o)
        dq, dk, dv = (_empty(t, t.shape[0], seqs.total) for t in (q, k, v))
        if seqs.total:
            a = _attention_args(q, k, v, o, lse, seqs, causal, scale)
            delta = torch.empty(q.shape[0], q.shape[1], device=q.device)
            a.d_o, a.d_q, a.d_k, a.d_v, a.delta = _tensor(d_o), _tensor(dq), _tensor(dk), _tensor(dv), delta.data_ptr()
            _launch_tiles("taco_attention_backward", a, seqs, q.device)
        return dq, dk, dv, None, None, None


def attention(q, k, v, sequences, causal=True, scale=None, return_lse=False, out=None):
    """softmax(scale q k^T) v inside each of `sequences` (a Packed): q [T, heads, dim], k and v [T, kv_heads, dim] with heads a multiple of kv_heads (query head h
    reads key-value head h // (heads // kv_heads)); T >= sequences.total.  causal: a token sees its own sequence up to itself, else all of it.
    scale: 1 / sqrt(dim).  -> [T, heads, dim]; with return_lse also log sum exp of the scaled scores, float32 [T, heads] (without gradient).
    A token that is hidden has no influence, even where it holds NaN or infinities, forward and backward.  Rows behind the last sequence: zero in new
    tensors and in gradients, untouched in `out` (which cannot be given where a gradient is recorded).
    Strides: any, as long as `dim` is contiguous and rows are multiples of 16 bytes; other layouts are copied first."""
    device, _ = _check_rows([("q", q), ("k", k), ("v", v)], "attention")
    _need(k.shape == v.shape and k.shape[0] == q.shape[0], f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}: the same tokens, and k and v alike, expected")
    _need(k.shape[1] > 0 and q.shape[1] > 0 and q.shape[1] % k.shape[1] == 0, f"{q.shape[1]} query heads cannot share {k.shape[1]} key-value heads")
    _need(isinstance(sequences, Packed), "sequences: a Packed expected")
    _need(sequences.device == device, f"q is on {device}, the sequences' work lists are on {sequences.device}")
    _need(sequences.total <= q.shape[0], f"{q.shape[0]} rows hold no {sequences.total} tokens")
    scale = _scale(scale, q.shape[2])
    _need(0 < scale < math.inf, f"scale {scale}: positive and finite")
    grad = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    if out is not None:
        _need(not grad, "out= cannot be given where a gradient is recorded")
        _need(out.shape == q.shape and out.dtype == q.dtype and out.device == device and _usable(out) is out, "out: q's shape, dtype and device, rows of whole 16-byte chunks")
    o, lse = _Attention.apply(q, k, v, sequences, causal, scale) if grad else _attention_forward(q, k, v, sequences, causal, scale, out)[3:]
    return (o, lse) if return_lse else o


# ---- attention of one token over a paged cache -------------------------------------------------------------------------------------

def attention_step(q, k, v, k_pages, v_pages, page_table, lengths, scale=None, out=None):
    """One new token per row over a paged key-value cache, which it joins.
    q [rows, heads, dim]; k, v [rows, kv_heads, dim]: the new token's; k_pages, v_pages [pages, page_size, kv_heads, dim] (any strides with `dim` contiguous,
    so a [pages, kv_heads, page_size, dim] cache is passed transposed); page_table int32 [rows, width]; lengths int32 [rows]: tokens in each row's cache
    BEFORE the call.  Token t of row b is page page_table[b, t // page_size], slot t % page_size.  The new token is written as token lengths[b] and
    attended too; lengths itself is the caller's to advance.  k = v = None: the cache is read as it is (a row of length 0 gives zeros).
    Rows may share pages that they only read.  A row whose length is negative or has no room in its table, or that reads a page number outside the cache,
    gives NaN; nothing else is touched.  -> [rows, heads, dim] (`out` if given).  No gradient."""
    named = [("q", q)] + ([("k", k), ("v", v)] if k is not None else [])
    _need((k is None) == (v is None), "k and v: both or none")
    device, code = _check_rows(named, "attention_step")
    B, H, d = q.shape
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        _need(t.dim() == 4 and t.shape[3] == d, f"{name} of shape {tuple(t.shape)}: [pages, page_size, kv_heads, {d}] expected")
        _need(t.dtype == q.dtype and t.device == device, f"{name} is {t.dtype} on {t.device}, q is {q.dtype} on {device}")
        size = t.element_size()
        if t.stride(3) != 1 or t.data_ptr() % 16 or any(t.shape[i] > 1 and (t.stride(i) * size % 16 or t.stride(i) < d) for i in range(3)):
            raise _lib.TacoError(f"{name}: rows of whole 16-byte chunks expected (strides {t.stride()})")
    P, page, Hk, _ = k_pages.shape
    _need(v_pages.shape == k_pages.shape and P > 0 and page > 0, f"k_pages {tuple(k_pages.shape)}, v_pages {tuple(v_pages.shape)}: alike and not empty expected")
    _need(Hk > 0 and H > 0 and H % Hk == 0, f"{H} query heads cannot share {Hk} key-value heads")
    _need(k is None or k.shape == v.shape == (B, Hk, d), f"k and v: [{B}, {Hk}, {d}] expected")
    for name, t, dim in (("page_table", page_table, 2), ("lengths", lengths, 1)):
        _need(t.dtype == torch.int32 and t.device == device and t.dim() == dim and t.shape[0] == B, f"{name}: int32 on {device}, {dim} dimensions, {B} rows expected")
        _need(t.shape[-1] <= 1 or t.stride(-1) == 1, f"{name}: contiguous rows expected")
    _need(page_table.shape[1] > 0, "page_table: at least one page per row")
    _no_grad((q, k, v, k_pages, v_pages), "attention_step")
    scale = _scale(scale, d)
    _need(0 < scale < math.inf, f"scale {scale}: positive and finite")
    if out is None:
        out = torch.empty(B, H, d, dtype=q.dtype, device=device)
    else:
        _need(out.shape == q.shape and out.dtype == q.dtype and out.device == device and _usable(out) is out, "out: q's shape, dtype and device, rows of whole 16-byte chunks")
    if B == 0:
        return out
    q = _usable(q)
    a = AttentionStepArgs()
    a.q, a.o = _tensor(q), _tensor(out)
    if k is not None:
        k, v = _usable(k), _usable(v)
        a.k_new, a.v_new = _tensor(k), _tensor(v)
    a.k_pages, a.v_pages = k_pages.data_ptr(), v_pages.data_ptr()

    def strides(t):         # (the stride of a dimension of one is never used)
        return [t.stride(i) if t.shape[i] > 1 else d for i in range(3)]
    a.k_page_stride, a.k_token_stride, a.k_head_stride = strides(k_pages)
    a.v_page_stride, a.v_token_stride, a.v_head_stride = strides(v_pages)
    a.table, a.table_stride, a.lengths = page_table.data_ptr(), page_table.stride(0), lengths.data_ptr()
    a.rows, a.table_width, a.num_pages, a.page_size = B, page_table.shape[1], P, page
    a.heads, a.kv_heads, a.dim, a.dtype, a.scale = H, Hk, d, code, scale
    need = load().taco_attention_step_workspace_bytes(C.byref(a))
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
    _call("taco_attention_step", a, device)
    return out


# ---- linear attention --------------------------------------------------------------------------------------------------------------

def _linear_args(q, k, v, log_decay, seqs, scale, products):
    a = LinearArgs()
    a.q, a.k, a.v = _tensor(q), _tensor(k), _tensor(v)
    a.log_decay = log_decay.data_ptr()
    segments, first, count = seqs._segments(q.shape[1] * products)
    a.segments, a.first_segment, a.n_segments, a.n_sequences = segments.data_ptr(), first.data_ptr(), count, len(seqs)
    a.heads, a.dim, a.dtype, a.scale = q.shape[1], q.shape[2], _DTYPES[q.dtype], scale
    return a


def _linear_workspace(a, backward, device):
    need = load().taco_linear_attention_workspace_bytes(C.byref(a), 1 if backward else 0)
    ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    a.workspace, a.workspace_bytes = (ws.data_ptr(), need) if need else (None, 0)
    return ws


def _linear_forward(q, k, v, log_decay, state, seqs, scale):
    q, k, v = _usable(q), _usable(k), _usable(v)
    o = _empty(q, q.shape[0], seqs.total)
    last = torch.empty(len(seqs), q.shape[1], q.shape[2], q.shape[2], device=q.device)
    if not seqs.total:              # no token: the states stay as they are
        last.zero_() if state is None else last.copy_(state)
    else:
        a = _linear_args(q, k, v, log_decay, seqs, scale, 1)
        a.o, a.state0, a.state_last = _tensor(o), state.data_ptr() if state is not None else None, last.data_ptr()
        ws = _linear_workspace(a, False, q.device)
        _call("taco_linear_attention", a, q.device)
        del ws
    return q, k, v, o, last


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, seqs, scale):
        q, k, v, o, last = _linear_forward(q, k, v, log_decay, state, seqs, scale)
        ctx.save_for_backward(q, k, v, log_decay, state)
        ctx.rest = seqs, scale
        ctx.set_materialize_grads(False)
        return o, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_o, d_last):
        q, k, v, log_decay, state = ctx.saved_tensors
        seqs, scale = ctx.rest
        d_o = torch.zeros_like(q) if d_o is None else _usable(d_o)
        dq, dk, dv = (_empty(t, t.shape[0], seqs.total) for t in (q, k, v))
        d_state = torch.empty_like(state) if state is not None and ctx.needs_input_grad[4] else None
        if not seqs.total:
            if d_state is not None:
                d_state.zero_() if d_last is None else d_state.copy_(d_last)
        else:
            a = _linear_args(q, k, v, log_decay, seqs, scale, 3)
            if d_last is not None:
                d_last = d_last.contiguous()
                a.d_state_last = d_last.data_ptr()
            a.state0, a.d_state0 = state.data_ptr() if state is not None else None, d_state.data_ptr() if d_state is not None else None
            a.d_o, a.d_q, a.d_k, a.d_v = _tensor(d_o), _tensor(dq), _tensor(dk), _tensor(dv)
            ws = _linear_workspace(a, True, q.device)
            _call("taco_linear_attention_backward", a, q.device)
            del ws
        return dq, dk, dv, None, d_state, None, None


def _check_decay(log_decay, heads, device):
    _need(log_decay.dtype == torch.float32 and log_decay.shape == (heads,) and log_decay.device == device, f"log_decay: float32 [{heads}] on {device} expected")
    if torch.is_grad_enabled() and log_decay.requires_grad:
        raise _lib.TacoError("log_decay has no gradient: the decays are constants of the model")
    return log_decay.contiguous()


def linear_attention(q, k, v, log_decay, sequences, state=None, scale=None):
    """S_t = exp(log_decay[head]) S_{t-1} + k_t v_t^T, o_t = scale * q_t S_t inside each of `sequences` (a Packed): q, k, v [T, heads, dim], log_decay float32 [heads]
    (<= 0 in earnest; -inf: only the token itself), state float32 [sequences, heads, dim, dim] (key dimension first) or None: the states to begin with.
    scale: 1 / sqrt(dim).  -> (o [T, heads, dim], the states behind the last tokens, float32).  Gradients for q, k, v and state.
    In float16 the states have to stay inside float16's range (65 504), which their product with q goes through.  A later token has no influence on an
    earlier output, even where it holds NaN or infinities."""
    device, _ = _check_rows([("q", q), ("k", k), ("v", v)], "linear_attention")
    _need(q.shape == k.shape == v.shape and q.shape[1] > 0, f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}: alike expected")
    _need(isinstance(sequences, Packed), "sequences: a Packed expected")
    _need(sequences.device == device, f"q is on {device}, the sequences' work lists are on {sequences.device}")
    _need(sequences.total <= q.shape[0], f"{q.shape[0]} rows hold no {sequences.total} tokens")
    H, d = q.shape[1:]
    log_decay = _check_decay(log_decay, H, device)
    if state is not None:
        _need(state.shape == (len(sequences), H, d, d) and state.dtype == torch.float32 and state.device == device, f"state: float32 [{len(sequences)}, {H}, {d}, {d}] on {device} expected")
        state = state.contiguous()
    scale = _scale(scale, d)
    _need(scale != 0 and math.isfinite(scale), f"scale {scale}: finite and not 0")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, state)):
        return _Linear.apply(q, k, v, log_decay, state, sequences, scale)
    return _linear_forward(q, k, v, log_decay, state, sequences, scale)[3:]


def linear_attention_step(q, k, v, log_decay, state, reset=None, scale=None, out=None):
    """One token per row of linear_attention: q, k, v [rows, heads, dim]; state float32 [rows, heads, dim, dim], contiguous, updated in place; reset [rows] (bool,
    uint8, int32 or int64, e.g. env.reset_buf): rows that begin anew, whatever their state holds.  -> [rows, heads, dim] (`out` if given).  No gradient."""
    device, code = _check_rows([("q", q), ("k", k), ("v", v)], "linear_attention_step")
    B, H, d = q.shape
    _need(q.shape == k.shape == v.shape and H > 0, f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}: alike expected")
    log_decay = _check_decay(log_decay, H, device)
    _need(state.shape == (B, H, d, d) and state.dtype == torch.float32 and state.device == device and state.is_contiguous() and state.data_ptr() % 16 == 0,
          f"state: float32 [{B}, {H}, {d}, {d}] on {device}, contiguous and 16-byte aligned, expected")
    _need(reset is None or reset.dtype in (torch.bool, torch.uint8, torch.int32, torch.int64) and reset.shape == (B,) and reset.device == device,
          f"reset: bool, uint8, int32 or int64 [{B}] on {device} expected")
    _no_grad((q, k, v, state), "linear_attention_step")
    scale = _scale(scale, d)
    _need(scale != 0 and math.isfinite(scale), f"scale {scale}: finite and not 0")
    if out is None:
        out = torch.empty(B, H, d, dtype=q.dtype, device=device)
    else:
        _need(out.shape == q.shape and out.dtype == q.dtype and out.device == device and _usable(out) is out, "out: q's shape, dtype and device, rows of whole 16-byte chunks")
    if B == 0:
        return out
    q, k, v = _usable(q), _usable(k), _usable(v)
    a = LinearStepArgs()
    a.q, a.k, a.v, a.o = _tensor(q), _tensor(k), _tensor(v), _tensor(out)
    a.log_decay, a.state = log_decay.data_ptr(), state.data_ptr()
    if reset is not None:
        reset = reset.contiguous()
        a.reset, a.reset_bytes = reset.data_ptr(), reset.element_size()
    a.rows, a.heads, a.dim, a.dtype, a.scale = B, H, d, code, scale
    _call("taco_linear_attention_step", a, device)
    return out
