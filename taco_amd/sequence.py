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
current stream of the tensors' device, nothing synchronises, and every call gives the same bits each time.  There is no torch fallback, no forward-mode derivative
and no second derivative: what asks for one is refused.

HIP graphs: call once eagerly before capturing (the work lists are uploaded at the first call with a given number of heads), keep the Packed alive as long as
the graph, and capture a backward pass only while no eager autograd graph of the same leaf tensors is alive: torch then waits for the eager graph's stream
inside the capture, which it does not survive.
"""
import ctypes as C
import functools
import math

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _lib

ABI_VERSION = 2
EXPORTS = ["taco_sequence_abi_version", "taco_sequence_source_hash", "taco_sequence_last_error", "taco_attention", "taco_attention_backward",
           "taco_attention_step_workspace_bytes", "taco_attention_step", "taco_linear_attention_workspace_bytes", "taco_linear_attention",
           "taco_linear_attention_backward", "taco_linear_attention_step"]
_FEW_SHORT = 1024       # workgroups of sequences of at most 64 tokens (four a CU) that still join the launch of the 128-row tiles (measured in Packed._tiles, on one shape)
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


class Tensor(C.Structure):
    """struct taco_seq_tensor"""
    _fields_ = [("ptr", C.c_void_p), ("token_stride", C.c_int64), ("head_stride", C.c_int64)]


class AttentionArgs(C.Structure):
    """struct taco_attention_args"""
    _fields_ = [("q", Tensor), ("k", Tensor), ("v", Tensor), ("o", Tensor), ("lse", C.c_void_p), ("tiles", C.c_void_p), ("key_tiles", C.c_void_p),
                ("n_tiles", C.c_int32), ("tile_rows", C.c_int32), ("whole", C.c_int32), ("heads", C.c_int32), ("kv_heads", C.c_int32), ("dim", C.c_int32), ("dtype", C.c_int32),
                ("causal", C.c_int32), ("scale", C.c_float), ("d_o", Tensor), ("d_q", Tensor), ("d_k", Tensor), ("d_v", Tensor), ("delta", C.c_void_p),
                ("parts", C.c_int32), ("partial", C.c_void_p)]


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


def _call(f, args, device):
    """an entry point on the current stream of the tensors' device"""
    if torch.cuda.current_device() == device.index:
        rc = f(C.byref(args), _lib.stream_ptr(device))
    else:                                       # a launch goes to the current device: make it the tensors'
        with torch.cuda.device(device):
            rc = f(C.byref(args), _lib.stream_ptr(device))
    if rc != 0:
        raise _lib.TacoError(f"libtaco_sequence: status {rc}: {load().taco_sequence_last_error().decode()}")


# what a call writes into a caller's tensor is a change in place for autograd too: a graph that has saved it refuses to run backward through it
_written = torch.autograd.graph.increment_version


# ---- checks shared by the calls (messages are made where a check fails: the host side of a call is most of a short one's time) ---------

def _check_rows(what, q, *others):
    """q and (name, tensor) pairs: [rows, heads, dim] tensors of one supported dtype on one HIP device -> (device, dtype code)"""
    device, dtype, shape = q.device, q.dtype, q.shape
    if device.type != "cuda":
        raise _lib.TacoError(f"{what} runs on an MI355X: q has to be on a cuda:N (HIP) device")
    code = _DTYPES.get(dtype)
    if code is None:
        raise _lib.TacoError(f"{what}: {dtype} is not supported (float32, float16, bfloat16)")
    if len(shape) != 3:
        raise ValueError(f"q of shape {tuple(shape)}: [tokens, heads, dim] expected")
    d = shape[2]
    for name, t in others:
        if t.dtype != dtype or t.device != device:
            raise ValueError(f"{name} is {t.dtype} on {t.device}, q is {dtype} on {device}")
        if len(t.shape) != 3 or t.shape[2] != d:
            raise ValueError(f"{name} of shape {tuple(t.shape)}: [tokens, heads, {d}] expected")
    if d % 8 or not 8 <= d <= 128:
        raise _lib.TacoError(f"{what}: head dimension {d} is not supported (a multiple of 8 from 8 to 128)")
    return device, code


def _usable(t):
    """`t` itself if the kernels can address it (rows of whole 16-byte chunks that do not overlap), else a contiguous copy"""
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
    (n, h, d), (ts, hs, ds), size = t.shape, t.stride(), t.element_size()
    if ds == 1 and t.data_ptr() % 16 == 0 and (h == 1 or hs * size % 16 == 0 and hs >= d) and (n == 1 or ts * size % 16 == 0 and d <= ts <= 1 << 21):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _tensor(t):
    """of a tensor that _usable() returned; the stride of a dimension of one is never used"""
    (n, h, d), (ts, hs, _) = t.shape, t.stride()
    return Tensor(t.data_ptr(), ts if n > 1 else h * d, hs if h > 1 else d)


def _check_out(out, q):
    if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or _usable(out) is not out:
        raise ValueError("out: q's shape, dtype and device, rows of whole 16-byte chunks")
    if out.requires_grad and torch.is_grad_enabled():       # (its graph would go on as if nothing had been written)
        raise _lib.TacoError("out requires a gradient: what is written into it has none")


def _scale(scale, dim, positive):
    if scale is None:
        return 1.0 / math.sqrt(dim)
    if isinstance(scale, torch.Tensor):
        if forward_ad._current_level >= 0:
            _no_tangent("the scale", scale)
        if scale.requires_grad and torch.is_grad_enabled():
            raise _lib.TacoError("the scale has no gradient: give its value, or multiply q by it")
    scale = float(scale)
    if not math.isfinite(scale) or scale == 0 or (positive and scale < 0):
        raise ValueError(f"scale {scale}: {'positive and finite' if positive else 'finite and not 0'}")
    return scale


def _no_grad(tensors, what):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise _lib.TacoError(f"{what} has no gradient: call it under torch.no_grad(), or use the form over whole sequences")


def _no_tangent(what, *tensors):
    """a dual tensor does not require a gradient: without this its tangent would be lost, and the result count as constant"""
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise _lib.TacoError(f"{what} has no forward-mode derivative")


def _check_packed(seqs, device, rows):
    if not isinstance(seqs, Packed):
        raise ValueError("sequences: a Packed expected")
    if seqs.device != device:
        raise ValueError(f"q is on {device}, the sequences' work lists are on {seqs.device}")
    if seqs.total > rows:
        raise ValueError(f"{rows} rows hold no {seqs.total} tokens")


class Packed:
    """Sequences behind one another in a tensor's first dimension: sequence i is rows [starts[i], starts[i] + lengths[i]).  `lengths`: non-negative whole numbers
    on the host (a list, an array, a CPU tensor); a device tensor is copied, which blocks.  Rows behind the last sequence may exist; no call reads them.
    Keeps the work lists of the kernels on `device`, made at the first call that needs them."""

    def __init__(self, lengths, device):
        n = lengths.detach().cpu().numpy() if isinstance(lengths, torch.Tensor) else np.asarray(lengths)
        if n.ndim != 1 or not (n.size == 0 or np.issubdtype(n.dtype, np.integer)):
            raise ValueError("lengths: one whole number per sequence expected")
        n = n.astype(np.int64)
        if (n < 0).any():
            raise ValueError("lengths: a sequence cannot have a negative length")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise _lib.TacoError("the sequence kernels run on an MI355X; device must be a cuda:N (HIP) device")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        limit = 2 ** 31 - 4096              # (a length of its own first: many such wrap around in their sum)
        self.lengths, self.starts, self.total = n, np.cumsum(n) - n, int(n.sum()) if (n < limit).all() else int(n.max())
        if self.total >= limit:
            raise ValueError(f"{self.total} tokens: fewer than 2^31 - 4096 are supported")
        self._lists = {}
        self._wide_tiles = int((-(-n[n > 64] // 128)).sum())
        self._short = int(np.count_nonzero((n > 0) & (n <= 64)))
        self._longest, self._pairs = int(n.max(initial=0)), float((n[n > 64].astype(np.float64) ** 2).sum())

    def __len__(self):
        return len(self.lengths)

    def _kept(self, key, make):
        """work list `key`: what make() returns, its arrays on the device"""
        got = self._lists.get(key)
        if got is None:
            if torch.cuda.is_current_stream_capturing():
                raise _lib.TacoError("the work list of these sequences is not on the device yet: make one call before capturing a graph")
            made = [torch.from_numpy(np.ascontiguousarray(t)).to(self.device) if isinstance(t, np.ndarray) else t for t in make()]
            got = self._lists[key] = (made, _lib.stream_ptr(self.device).value)
        elif got[1] != _lib.stream_ptr(self.device).value and not torch.cuda.is_current_stream_capturing():
            for t in got[0]:                    # another stream than the lists' own: their memory is not given away before its work is done
                if isinstance(t, torch.Tensor):
                    t.record_stream(torch.cuda.current_stream(self.device))
        return got[0]

    def _wide(self, heads):
        """whether there are tiles of 128 rows: if those alone fill the CUs"""
        return self._wide_tiles * heads >= 256

    def _tiles(self, heads):
        """[(tile rows, tiles, key tiles, count, how many of them at the end are whole sequences)].  A tile of 128 rows shares its loads between four wavefronts;
        sequences of at most 64 tokens would leave half of it idle, and where all tiles together do not fill the CUs, smaller ones spread the work.  Sequences
        of at most 32 tokens are a tile each.  A few short sequences beside many long ones take a 128-row tile each all the same: launches of their own would
        run on some CUs after the others (100 sequences of 65 to 200 tokens, 8 heads of 128 over 2, and 30 of up to 64, forward and backward: bf16 283 -> 229 us,
        float32 1.03 -> 0.79 ms; with 120 short ones 323 -> 313 us; with 250 they would cost 351 -> 388)."""
        wide = self._wide(heads)
        few = wide and self._short * heads <= _FEW_SHORT
        key = "wide tiles only" if few else "wide tiles" if wide else "tiles"

        def tiles(rows, which):
            which = np.flatnonzero(which)
            n = -(-self.lengths[which] // rows)
            of = np.repeat(which, n)
            first = (np.arange(len(of)) - np.repeat(np.cumsum(n) - n, n)) * rows
            t = np.stack([self.starts[of], self.lengths[of], first, np.zeros_like(first)], 1).astype(np.int32)
            return t[np.argsort(-np.minimum(first + rows, self.lengths[of]), kind="stable")], t[np.argsort(first - self.lengths[of], kind="stable")]

        def make():
            big, short = (self.lengths > (0 if few else 64)) & wide, self.lengths <= 32
            large, some, whole = tiles(128, big), tiles(32, ~big & ~short), tiles(32, short & ~big & (self.lengths > 0))
            small = [np.concatenate(x) for x in zip(some, whole)]
            return (128, *large, len(large[0]), 0, 32, *small, len(small[0]), len(whole[0]))
        got = self._kept(key, make)
        return [got[i:i + 5] for i in (0, 5) if got[i + 3]]

    def _parts(self, heads, group, causal):
        """Into how many parts the backward's second launch shares out a group's query heads: few enough that their partial sums' way through memory stays small, but
        so many that the longest sequence's first tile of keys, which sees all its queries, takes no longer than a CU's share of everything.  (Only tiles of 128
        rows are: with others alone there is one part, and no memory for sums.)"""
        if not self._wide(heads):
            return 1
        share = self._pairs * (0.5 if causal else 1.0) * heads / 128 / 256
        for parts in range(1, group + 1):
            if group % parts == 0 and self._longest * (group // parts) <= share:
                return parts
        return group

    def _segments(self, work):
        """(segments, first segment of each sequence, count) for `work` = heads x products: workgroups for each segment, one to a CU.  Fewer, longer segments leave CUs
        idle; each cut costs a second reading of its k and v and the state's way through memory and back.  Of some lengths (at least 256 tokens; sequences
        are cut into equal pieces) the one with the least estimate is taken, in tokens of a CU's time: the longest segment if all run at once, else a CU's
        share and half the longest; a third for a token that is read again; 160 for a state (six sequences of 28 700 tokens, 16 heads: 213 us in 15
        segments, 241 in 34).  Both weights come from that one shape, bf16 heads of 128; a state's goes with the square of the head size and neither that nor the type
        enters: elsewhere the estimate chooses a working cut, not always the best."""
        got = self._lists.get(("segments", work))
        if got is not None:
            return self._kept(("segments", work), None)

        def pieces(size):
            return np.maximum(-(-self.lengths // size), 1)

        def estimate(size):
            n = pieces(size)
            longest, share = (self.lengths / n).max(initial=0), self.total * work / 256
            again = (self.lengths * (n - 1) / n).sum() / 3 + 160 * n[n > 1].sum()
            return (longest if n.sum() * work <= 256 else share + longest / 2) + again * work / 256

        def make():
            uncut = max(self._longest, 256)
            sizes = {max(256, -(-int(self.total * work / (256 * rounds)) // 64) * 64) for rounds in (0.75, 0.9, 1, 1.2, 1.5, 1.75, 2, 2.5, 3, 4)}
            n = pieces(min([uncut] + sorted(sizes, reverse=True), key=estimate))
            if n.sum() > len(n) and len(n) * work > 65535:      # (the joining launch's limit; so many sequences fill the CUs by themselves)
                n = np.ones_like(n)
            first = np.concatenate([[0], np.cumsum(n)])
            of = np.repeat(np.arange(len(n)), n)
            index = np.arange(len(of)) - first[of]
            step = np.where(n[of] > 1, -(-self.lengths[of] // (n[of] * 64)) * 64, self.lengths[of])
            at = index * step
            cols = [of, self.starts[of], self.lengths[of], at, np.minimum(step, self.lengths[of] - at), index, index * 0, index * 0]
            return [np.stack(cols, 1).astype(np.int32).reshape(-1, 8), first.astype(np.int32), len(of)]
        return self._kept(("segments", work), make)


# ---- attention over packed sequences -----------------------------------------------------------------------------------------------

def _attention_args(q, k, v, o, lse, seqs, causal, scale):
    heads, dim = q.shape[1], q.shape[2]
    return AttentionArgs(_tensor(q), _tensor(k), _tensor(v), _tensor(o), lse.data_ptr(), None, None, 0, 0, 0, heads, k.shape[1], dim, _DTYPES[q.dtype], 1 if causal else 0, scale)


def _launch_tiles(a, seqs, device, backward):
    lib = load()
    for rows, tiles, key_tiles, count, whole in seqs._tiles(a.heads):
        a.tile_rows, a.tiles, a.key_tiles, a.n_tiles = rows, tiles.data_ptr(), key_tiles.data_ptr(), count
        if not backward:
            _call(lib.taco_attention, a, device)
            continue
        if a.dtype == 0 and a.dim > 96:     # (float32 rows this wide: no form for whole sequences)
            whole = 0
        a.n_tiles = count - whole           # (whole sequences have a launch of their own)
        if a.n_tiles:
            _call(lib.taco_attention_backward, a, device)
        if whole:
            skip = (count - whole) * C.sizeof(C.c_int32 * 4)
            a.tiles, a.key_tiles, a.n_tiles, a.whole = a.tiles + skip, a.key_tiles + skip, whole, 1
            _call(lib.taco_attention_backward, a, device)
            a.whole = 0


def _empty(shape, total, dtype, device):
    """uninitialised [rows, ...]; rows behind the last sequence are zero"""
    t = torch.empty(shape, dtype=dtype, device=device)
    if shape[0] > total:
        t[total:].zero_()
    return t


class _OnceOnly(torch.autograd.Function):
    """The last `count` tensors, as functions of those before them whose derivative is refused: gradients that were asked for with create_graph, which torch would
    otherwise take for constants wherever the upstream gradient is one."""
    @staticmethod
    def forward(ctx, count, *tensors):
        return tuple(t.clone() for t in tensors[-count:])

    @staticmethod
    def backward(ctx, *_):
        raise _lib.TacoError("the sequence operators have no second derivative")


def _first_derivative(f):
    """of a Function's backward pass: it runs unrecorded, and what it returns cannot be differentiated again"""
    @functools.wraps(f)
    def backward(ctx, *upstream):
        with torch.no_grad():
            grads = f(ctx, *upstream)
        if not torch.is_grad_enabled():
            return grads
        at = [i for i, g in enumerate(grads) if g is not None]
        if at:
            of = [t for t in (*ctx.saved_tensors, *upstream) if t is not None]
            grads = list(grads)
            for i, g in zip(at, _OnceOnly.apply(len(at), *of, *(grads[i] for i in at))):
                grads[i] = g
        return tuple(grads)
    return backward


def _attention_forward(q, k, v, seqs, causal, scale, out):
    """(q, k and v as _usable returned them)"""
    total, device = seqs.total, q.device
    o = _empty(q.shape, total, q.dtype, device) if out is None else out
    lse = _empty(q.shape[:2], total, torch.float32, device)
    if out is not None:
        _written(out)
    if total:
        _launch_tiles(_attention_args(q, k, v, o, lse, seqs, causal, scale), seqs, device, False)
    return o, lse


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, seqs, causal, scale):
        o, lse = _attention_forward(q, k, v, seqs, causal, scale, None)
        ctx.save_for_backward(q, k, v, o, lse)
        ctx.rest = seqs, causal, scale
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return o, lse

    @staticmethod
    @_first_derivative
    def backward(ctx, d_o, _):
        if d_o is None:
            return (None,) * 6
        q, k, v, o, lse = ctx.saved_tensors
        seqs, causal, scale = ctx.rest
        d_o = _usable(d_o)
        dq, dk, dv = (_empty(t.shape, seqs.total, t.dtype, t.device) for t in (q, k, v))
        if seqs.total:
            a = _attention_args(q, k, v, o, lse, seqs, causal, scale)
            delta = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
            a.d_o, a.d_q, a.d_k, a.d_v, a.delta = _tensor(d_o), _tensor(dq), _tensor(dk), _tensor(dv), delta.data_ptr()
            H, Hk, d = q.shape[1], k.shape[1], q.shape[2]
            a.parts = seqs._parts(H, H // Hk, causal)
            if a.parts > 1:
                wide = seqs._tiles(H)[0][3]
                partial = torch.empty((wide * 128, Hk, a.parts, 2, -(-d // 32) * 32), dtype=torch.float32, device=q.device)
                a.partial = partial.data_ptr()
            _launch_tiles(a, seqs, q.device, True)
        return dq, dk, dv, None, None, None


def attention(q, k, v, sequences, causal=True, scale=None, return_lse=False, out=None):
    """softmax(scale q k^T) v inside each of `sequences` (a Packed): q [T, heads, dim], k and v [T, kv_heads, dim] with heads a multiple of kv_heads (query head h
    reads key-value head h // (heads // kv_heads)); T >= sequences.total.  causal: a token sees its own sequence up to itself, else all of it.
    scale: 1 / sqrt(dim).  -> [T, heads, dim]; with return_lse also log sum exp of the scaled scores, float32 [T, heads] (without gradient).
    A token that is hidden has no influence, even where it holds NaN or infinities, forward and backward; a token whose scores are all -inf gets zeros.  Rows behind the last sequence: zero in new
    tensors and in gradients, untouched in `out` (which cannot be given where a gradient is recorded, and must not overlap q, k or v).
    Strides: any, as long as `dim` is contiguous and rows are multiples of 16 bytes; other layouts are copied first."""
    if forward_ad._current_level >= 0:
        _no_tangent("attention", q, k, v, out)
    device, _ = _check_rows("attention", q, ("k", k), ("v", v))
    (T, H, d), Hk = q.shape, k.shape[1]
    if k.shape != v.shape or k.shape[0] != T:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}: the same tokens, and k and v alike, expected")
    if not Hk or not H or H % Hk:
        raise ValueError(f"{H} query heads cannot share {Hk} key-value heads")
    _check_packed(sequences, device, T)
    scale = _scale(scale, d, True)
    grad = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    if out is not None:
        if grad:
            raise ValueError("out= cannot be given where a gradient is recorded")
        _check_out(out, q)
    q, k, v = _usable(q), _usable(k), _usable(v)
    o, lse = _Attention.apply(q, k, v, sequences, causal, scale) if grad else _attention_forward(q, k, v, sequences, causal, scale, out)
    return (o, lse) if return_lse else o


# ---- attention of one token over a paged cache -------------------------------------------------------------------------------------

_step_workspace = {}        # bytes of taco_attention_step's workspace by shape


def _check_pages(name, t, q):
    """-> its page, token and head stride (of a dimension of one: any that pass the checks)"""
    shape, stride, d = t.shape, t.stride(), q.shape[2]
    if t.dtype != q.dtype or t.device != q.device:
        raise ValueError(f"{name} is {t.dtype} on {t.device}, q is {q.dtype} on {q.device}")
    if len(shape) != 4 or shape[3] != d:
        raise ValueError(f"{name} of shape {tuple(shape)}: [pages, page_size, kv_heads, {d}] expected")
    unit = 16 // t.element_size()
    out = [stride[i] if shape[i] > 1 else d for i in range(3)]
    if stride[3] != 1 or t.data_ptr() % 16 or any(s % unit or s < d for s in out):
        raise _lib.TacoError(f"{name}: rows of whole 16-byte chunks expected (strides {stride})")
    return out


def attention_step(q, k, v, k_pages, v_pages, page_table, lengths, scale=None, out=None):
    """One new token per row over a paged key-value cache, which it joins.
    q [rows, heads, dim]; k, v [rows, kv_heads, dim]: the new token's; k_pages, v_pages [pages, page_size, kv_heads, dim] (any strides with `dim` contiguous,
    so a [pages, kv_heads, page_size, dim] cache is passed transposed); page_table int32 [rows, width]; lengths int32 [rows]: tokens in each row's cache
    BEFORE the call.  Token t of row b is page page_table[b, t // page_size], slot t % page_size.  The new token is written as token lengths[b] and
    attended too; lengths itself is the caller's to advance.  k = v = None: the cache is read as it is (a row of length 0 gives zeros).
    Rows may share pages that they only read; the slot a token is written to has to be named once, by one row, and rows that take no part get a length of -1.
    A row whose length is negative or has no room in its table, or that reads a page number outside the cache, gives NaN; what other rows hold is not touched
    (its own token still joins the cache if that has a page and a slot).  -> [rows, heads, dim] (`out` if given, which must not overlap the inputs).  No gradient."""
    if (k is None) != (v is None):
        raise ValueError("k and v: both or none")
    if forward_ad._current_level >= 0:
        _no_tangent("attention_step", q, k, v, k_pages, v_pages, out)
    device, code = _check_rows("attention_step", q) if k is None else _check_rows("attention_step", q, ("k", k), ("v", v))
    B, H, d = q.shape
    ks, vs = _check_pages("k_pages", k_pages, q), _check_pages("v_pages", v_pages, q)
    P, page, Hk, _ = k_pages.shape
    if v_pages.shape != k_pages.shape or not P or not page:
        raise ValueError(f"k_pages {tuple(k_pages.shape)}, v_pages {tuple(v_pages.shape)}: alike and not empty expected")
    if not Hk or not H or H % Hk:
        raise ValueError(f"{H} query heads cannot share {Hk} key-value heads")
    if k is not None and not k.shape == v.shape == (B, Hk, d):
        raise ValueError(f"k {tuple(k.shape)}, v {tuple(v.shape)}: [{B}, {Hk}, {d}] expected")
    for name, t, dim in (("page_table", page_table, 2), ("lengths", lengths, 1)):
        if t.dtype != torch.int32 or t.device != device or t.dim() != dim or t.shape[0] != B:
            raise ValueError(f"{name}: int32 on {device}, {dim} dimensions, {B} rows expected")
        if t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{name}: contiguous rows expected")
    width = page_table.shape[1]
    if not width:
        raise ValueError("page_table: at least one page per row")
    _no_grad((q, k, v, k_pages, v_pages), "attention_step")
    scale = _scale(scale, d, True)
    if out is None:
        out = torch.empty((B, H, d), dtype=q.dtype, device=device)
    else:
        _check_out(out, q)
    if not B:
        return out
    q = _usable(q)
    if H > 1 and q.stride(1) > 1 << 21:         # (a descriptor reaches over the heads of a row)
        q = q.contiguous()
    if k is None:
        new_k = new_v = Tensor()
    else:
        k, v = _usable(k), _usable(v)
        new_k, new_v = _tensor(k), _tensor(v)
    a = AttentionStepArgs(_tensor(q), _tensor(out), new_k, new_v, k_pages.data_ptr(), v_pages.data_ptr(), *ks, *vs, page_table.data_ptr(), page_table.stride(0),
                          lengths.data_ptr(), B, width, P, page, H, Hk, d, code, scale, None, 0)
    lib = load()
    shape = (B, H, Hk, d, width, page)
    need = _step_workspace.get(shape)
    if need is None:
        need = _step_workspace[shape] = lib.taco_attention_step_workspace_bytes(C.byref(a))
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
    _call(lib.taco_attention_step, a, device)
    _written((out,) if k is None else (out, k_pages, v_pages))
    return out


# ---- linear attention --------------------------------------------------------------------------------------------------------------

def _linear_args(q, k, v, log_decay, seqs, scale, products):
    heads, dim = q.shape[1], q.shape[2]
    segments, first, count = seqs._segments(heads * products)
    return LinearArgs(_tensor(q), _tensor(k), _tensor(v), Tensor(), log_decay.data_ptr(), None, None, segments.data_ptr(), first.data_ptr(), count, len(seqs),
                      heads, dim, _DTYPES[q.dtype], scale)


def _linear_workspace(a, seqs, backward, device):
    if a.n_segments == len(seqs):
        return None
    need = load().taco_linear_attention_workspace_bytes(C.byref(a), 1 if backward else 0)
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    a.workspace, a.workspace_bytes = ws.data_ptr(), need
    return ws


def _linear_forward(q, k, v, log_decay, state, seqs, scale):
    """(q, k and v as _usable returned them)"""
    o = _empty(q.shape, seqs.total, q.dtype, q.device)
    last = torch.empty((len(seqs), q.shape[1], q.shape[2], q.shape[2]), dtype=torch.float32, device=q.device)
    if not seqs.total:              # no token: the states stay as they are
        last.zero_() if state is None else last.copy_(state)
    else:
        a = _linear_args(q, k, v, log_decay, seqs, scale, 1)
        a.o, a.state0, a.state_last = _tensor(o), state.data_ptr() if state is not None else None, last.data_ptr()
        ws = _linear_workspace(a, seqs, False, q.device)
        _call(load().taco_linear_attention, a, q.device)
        del ws
    return o, last


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, seqs, scale):
        o, last = _linear_forward(q, k, v, log_decay, state, seqs, scale)
        ctx.save_for_backward(q, k, v, log_decay, state)
        ctx.rest = seqs, scale
        ctx.set_materialize_grads(False)
        return o, last

    @staticmethod
    @_first_derivative
    def backward(ctx, d_o, d_last):
        q, k, v, log_decay, state = ctx.saved_tensors
        seqs, scale = ctx.rest
        d_o = torch.zeros_like(q) if d_o is None else _usable(d_o)
        dq, dk, dv = (_empty(t.shape, seqs.total, t.dtype, t.device) for t in (q, k, v))
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
            ws = _linear_workspace(a, seqs, True, q.device)
            _call(load().taco_linear_attention_backward, a, q.device)
            del ws
        return dq, dk, dv, None, d_state, None, None


def _check_decay(log_decay, heads, device):
    if log_decay.dtype != torch.float32 or log_decay.shape != (heads,) or log_decay.device != device:
        raise ValueError(f"log_decay: float32 [{heads}] on {device} expected")
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise _lib.TacoError("log_decay has no gradient: the decays are constants of the model")
    return log_decay.contiguous()


def linear_attention(q, k, v, log_decay, sequences, state=None, scale=None):
    """S_t = exp(log_decay[head]) S_{t-1} + k_t v_t^T, o_t = scale * q_t S_t inside each of `sequences` (a Packed): q, k, v [T, heads, dim], log_decay float32 [heads]
    (<= 0 in earnest; -inf: only the token itself), state float32 [sequences, heads, dim, dim] (key dimension first) or None: the states to begin with.
    scale: 1 / sqrt(dim).  -> (o [T, heads, dim], the states behind the last tokens, float32).  Gradients for q, k, v and state.
    A later token has no influence on an earlier output, even where it holds NaN or infinities; a value that is not finite makes the outputs of its own chunk of
    64 tokens and the state NaN.  In float16 a growth (log_decay > 0) must leave v exp(64 log_decay) inside the type's range."""
    if forward_ad._current_level >= 0:
        _no_tangent("linear_attention", q, k, v, log_decay, state)
    device, _ = _check_rows("linear_attention", q, ("k", k), ("v", v))
    if not q.shape == k.shape == v.shape or not q.shape[1]:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}: alike expected")
    T, H, d = q.shape
    _check_packed(sequences, device, T)
    log_decay = _check_decay(log_decay, H, device)
    if state is not None:
        if state.shape != (len(sequences), H, d, d) or state.dtype != torch.float32 or state.device != device:
            raise ValueError(f"state: float32 [{len(sequences)}, {H}, {d}, {d}] on {device} expected")
        state = state.contiguous()
    scale = _scale(scale, d, False)
    q, k, v = _usable(q), _usable(k), _usable(v)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, state)):
        return _Linear.apply(q, k, v, log_decay, state, sequences, scale)
    return _linear_forward(q, k, v, log_decay, state, sequences, scale)


_RESET_BYTES = {torch.bool: 1, torch.uint8: 1, torch.int32: 4, torch.int64: 8}


def linear_attention_step(q, k, v, log_decay, state, reset=None, scale=None, out=None):
    """One token per row of linear_attention: q, k, v [rows, heads, dim]; state float32 [rows, heads, dim, dim], contiguous, updated in place; reset [rows] (bool,
    uint8, int32 or int64, e.g. env.reset_buf): rows that begin anew, whatever their state holds.  -> [rows, heads, dim] (`out` if given, which must not
    overlap the inputs).  No gradient."""
    if forward_ad._current_level >= 0:
        _no_tangent("linear_attention_step", q, k, v, log_decay, state, out)
    device, code = _check_rows("linear_attention_step", q, ("k", k), ("v", v))
    shape = q.shape
    B, H, d = shape
    if k.shape != shape or v.shape != shape or not H:
        raise ValueError(f"q {tuple(shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}: alike expected")
    log_decay = _check_decay(log_decay, H, device)
    if state.shape != (B, H, d, d) or state.dtype != torch.float32 or state.device != device or not state.is_contiguous() or state.data_ptr() % 16:
        raise ValueError(f"state: float32 [{B}, {H}, {d}, {d}] on {device}, contiguous and 16-byte aligned, expected")
    if reset is not None:
        if reset.dtype not in _RESET_BYTES or reset.shape != (B,) or reset.device != device:
            raise ValueError(f"reset: bool, uint8, int32 or int64 [{B}] on {device} expected")
        reset = reset.contiguous()
    _no_grad((q, k, v, state), "linear_attention_step")
    scale = _scale(scale, d, False)
    if out is None:
        out = torch.empty(shape, dtype=q.dtype, device=device)
    else:
        _check_out(out, q)
    if not B:
        return out
    q, k, v = _usable(q), _usable(k), _usable(v)
    a = LinearStepArgs(_tensor(q), _tensor(k), _tensor(v), _tensor(out), log_decay.data_ptr(), state.data_ptr(), None if reset is None else reset.data_ptr(),
                       0 if reset is None else _RESET_BYTES[reset.dtype], B, H, d, code, scale)
    _call(load().taco_linear_attention_step, a, device)
    _written((out, state))
    return out
