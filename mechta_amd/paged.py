"""Python mirror of the paged cache's C ABI (include/mechta_paged.h), over the same libmechta_kv.so.

Many sequences share one pool of pages: PagedKv keeps the pages, forks, copies, frees and compacts them, appends the new
tokens of a batch (rotating K and q) and attends over the pages; rotate() applies rotary positions alone. Every compute
call goes through the HIP library.
"""
import ctypes
from array import array

from mechta_amd import F16, F32, K, V, MkvError, lib as _mkv_lib  # noqa: F401

BF16 = 2

# every symbol include/mechta_paged.h declares
SYMBOLS = ["mpg_rope_freqs", "mpg_rope_turns", "mpg_rotate", "mpg_bytes", "mpg_create", "mpg_destroy", "mpg_set_stream", "mpg_sync",
           "mpg_len", "mpg_table", "mpg_free_pages", "mpg_pages", "mpg_reserve", "mpg_begin", "mpg_begin_shared", "mpg_set_len", "mpg_fork",
           "mpg_copy", "mpg_free", "mpg_compact", "mpg_append", "mpg_attend", "mpg_read_rows",
           "mpg_weights_bytes", "mpg_keep_weights", "mpg_weights", "mpg_weigh", "mpg_evict", "mpg_position"]

LAYOUTS = {"half": 0, "interleaved": 1}
SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "bands": 4}

_FORMATS = {}  # torch's element types, filled in on first use
_done = False


class _Rope(ctypes.Structure):
    _fields_ = [("dim", ctypes.c_int), ("layout", ctypes.c_int), ("scaling", ctypes.c_int), ("original", ctypes.c_int),
                ("base", ctypes.c_double), ("factor", ctypes.c_double), ("beta_fast", ctypes.c_double),
                ("beta_slow", ctypes.c_double), ("low", ctypes.c_double), ("high", ctypes.c_double),
                ("amplitude", ctypes.c_double)]


class _Turns(ctypes.Structure):
    _fields_ = [("turns", ctypes.c_double * 256), ("amplitude", ctypes.c_float), ("dim", ctypes.c_int),
                ("layout", ctypes.c_int)]


class _Config(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("layers", "q_heads", "kv_heads", "head_dim", "fmt", "pages", "page", "seqs",
                                            "ctx", "tokens")]


def lib():
    global _done
    L = _mkv_lib()
    if not _done:
        P, I, F, S, L64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_size_t, ctypes.c_int64
        R, T, C = ctypes.POINTER(_Rope), P, ctypes.POINTER(_Config)
        IP, DP = ctypes.POINTER(I), ctypes.POINTER(ctypes.c_double)
        sig = {
            "mpg_rope_freqs": ([R, DP, DP], I),
            "mpg_rope_turns": ([R, T], I),
            "mpg_rotate": ([T, I, I, I, I, P, L64, L64, P, P, L64, L64, P], I),
            "mpg_bytes": ([C], S),
            "mpg_create": ([ctypes.POINTER(P), C, P, R, P], I),
            "mpg_destroy": ([P], I),
            "mpg_set_stream": ([P, P], I),
            "mpg_sync": ([P], I),
            "mpg_len": ([P, I, IP], I),
            "mpg_table": ([P, I, IP, I], I),
            "mpg_free_pages": ([P, IP], I),
            "mpg_pages": ([P, I, I, ctypes.POINTER(P)], I),
            "mpg_reserve": ([P, I, P, P], I),
            "mpg_begin": ([P, I, P, P, IP], I),
            "mpg_begin_shared": ([P, I, P, P, IP], I),
            "mpg_set_len": ([P, I, I], I),
            "mpg_fork": ([P, I, P, P, P], I),
            "mpg_copy": ([P, I, P, P], I),
            "mpg_free": ([P, I, P], I),
            "mpg_compact": ([P, IP], I),
            "mpg_append": ([P, I, I, P, L64, L64, P, L64, L64, P, L64, L64, P, I], I),
            "mpg_attend": ([P, I, I, P, L64, L64, F, P, P, L64, L64, P], I),
            "mpg_read_rows": ([P, I, I, I, I, I, P], I),
            "mpg_weights_bytes": ([C, I], S),
            "mpg_keep_weights": ([P, I], I),
            "mpg_weights": ([P, I, ctypes.POINTER(P), ctypes.POINTER(L64), ctypes.POINTER(L64)], I),
            "mpg_weigh": ([P, I, I, P, L64, L64, F, P, F], I),
            "mpg_evict": ([P, I, P, P, I, I], I),
            "mpg_position": ([P, I, IP], I),
        }
        for name, (args, res) in sig.items():
            f = getattr(L, name)
            f.argtypes = args
            f.restype = res
        _done = True
    return L


def _check(rc):
    if rc < 0:
        raise MkvError(rc, lib().mkv_last_error().decode())
    return rc


def _ints(xs, n=None, what="list"):
    """A list of ints as an array and its address; the array is to live as long as that is used."""
    try:
        a = array("i", xs)
    except OverflowError:
        raise ValueError(f"{what} has entries past 32 bits") from None
    if n is not None and len(a) != n:
        raise ValueError(f"{what} has {len(a)} entries, {n} needed")
    return a, a.buffer_info()[0]


def _int(x, what):
    """x, refused where the C ABI's int does not hold it (ctypes would pass on its low 32 bits)."""
    if not -1 << 31 <= x < 1 << 31:
        raise ValueError(f"{what} {x} is past 32 bits")
    return x


def _config(layers, q_heads, kv_heads, head_dim, pages, page, seqs, ctx, fmt, tokens):
    c = _Config()
    for name, x in dict(layers=layers, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, fmt=fmt, pages=pages, page=page,
                        seqs=seqs, ctx=ctx, tokens=tokens).items():
        setattr(c, name, _int(x, name))
    return c


def _dtype(fmt):
    import torch
    return {F16: torch.float16, F32: torch.float32, BF16: torch.bfloat16}[fmt]


class Rope:
    """Rotary positions: the first `dim` elements of a head turn, in pairs (i, i + dim/2) ("half") or (2i, 2i + 1)
    ("interleaved"). scaling: "none", "linear", "ntk", "yarn" or "bands", by `factor`, with the context `original` that
    the model was trained on for the last two (include/mechta_paged.h has the formulas)."""

    def __init__(self, dim, layout="half", base=10000.0, scaling="none", factor=1.0, original=0, beta_fast=32.0,
                 beta_slow=1.0, low=1.0, high=4.0, amplitude=0.0):
        if layout not in LAYOUTS:
            raise ValueError(f"layout {layout!r}: one of {', '.join(LAYOUTS)}")
        if scaling not in SCALINGS:
            raise ValueError(f"scaling {scaling!r}: one of {', '.join(SCALINGS)}")
        self.c = _Rope(_int(dim, "dim"), LAYOUTS[layout], SCALINGS[scaling], _int(int(original), "original"), base, factor, beta_fast, beta_slow, low,
                       high, amplitude)
        self.dim = dim
        self._turns = _Turns()
        _check(lib().mpg_rope_turns(ctypes.byref(self.c), ctypes.byref(self._turns)))
        self._ptr = ctypes.addressof(self._turns)

    def __setstate__(self, state):  # copies and pickles go by the turns of their own
        self.__dict__.update(state)
        self._ptr = ctypes.addressof(self._turns)

    def freqs(self):
        """(turning speed of each pair in radians per position, amplitude)."""
        th, amp = (ctypes.c_double * max(self.dim // 2, 1))(), ctypes.c_double()
        _check(lib().mpg_rope_freqs(ctypes.byref(self.c), th, ctypes.byref(amp)))
        return list(th), amp.value


def _rows(t, heads, dim, dtype, device, what):
    """Checks a [rows, heads, dim] tensor whose last dimension is contiguous; returns its address and strides."""
    shape, stride = t.shape, t.stride()
    if t.dtype is dtype and t.device == device and len(shape) == 3 and shape[1] == heads and shape[2] == dim \
            and (stride[2] == 1 or dim == 1):
        return t.data_ptr(), stride[0], stride[1]
    if t.device != device:
        raise ValueError(f"{what} is on {t.device}, {device} needed")
    if t.dtype is not dtype:
        raise ValueError(f"{what} is {t.dtype}, {dtype} needed")
    if len(shape) != 3 or shape[1] != heads or shape[2] != dim:
        raise ValueError(f"{what} has shape {tuple(shape)}, (rows, {heads}, {dim}) needed")
    raise ValueError(f"the last dimension of {what} must be contiguous")


def rotate(x, pos, rope, out=None):
    """x [rows, heads, dim] (f16, bf16 or f32) rotated at the positions pos [rows] (int32), into `out` (may be x), on
    torch's current stream of x's device."""
    import torch
    dtype, device, shape = x.dtype, x.device, x.shape
    fmt = _FORMATS.get(dtype)
    if fmt is None:
        if x.is_floating_point() and not _FORMATS:
            _FORMATS.update({torch.float16: F16, torch.float32: F32, torch.bfloat16: BF16})
        fmt = _FORMATS.get(dtype)
        if fmt is None:
            raise ValueError(f"x is {dtype}: float16, bfloat16 or float32 needed")
    if len(shape) != 3:
        raise ValueError(f"x has shape {tuple(shape)}, (rows, heads, dim) needed")
    rows, heads, dim = shape
    if (rows | heads | dim) >> 31:
        raise ValueError(f"x of shape {tuple(shape)} is past 32 bits")
    if device.type != "cuda":
        raise ValueError("x must be a device tensor")
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    elif out.shape[:1] != shape[:1]:
        raise ValueError(f"out has shape {tuple(out.shape)}, x {tuple(shape)}")
    xp, xr, xh = _rows(x, heads, dim, dtype, device, "x")
    op, orow, oh = _rows(out, heads, dim, dtype, device, "out")
    if pos.device != device or pos.dtype is not torch.int32 or pos.shape != shape[:1] or not pos.is_contiguous():
        raise ValueError(f"pos must be {rows} contiguous int32 on {device}")
    stream = torch._C._cuda_getCurrentRawStream(device.index)
    if torch.cuda.current_device() == device.index:
        rc = lib().mpg_rotate(rope._ptr, fmt, rows, heads, dim, xp, xr, xh, pos.data_ptr(), op, orow, oh, stream)
    else:
        with torch.cuda.device(device):
            rc = lib().mpg_rotate(rope._ptr, fmt, rows, heads, dim, xp, xr, xh, pos.data_ptr(), op, orow, oh, stream)
    if rc:
        _check(rc)
    return out


class _Handle:
    """Owns an mpg_t*: the cache and every tensor over its pages hold it."""

    def __init__(self):
        self.ptr = ctypes.c_void_p()

    def close(self):
        if self.ptr:
            lib().mpg_destroy(self.ptr)
            self.ptr = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class PagedKv:
    """The paged cache of `layers` layers: `pages` pages of `page` positions for up to `seqs` sequences of up to `ctx`
    positions; batches of up to `tokens` new tokens. fmt: F16 or BF16 (pages, q, k, v, gate, out). windows: per layer the
    positions a token sees, itself included (0 or None: all). rope: what append() rotates by. weigh_last: the cache keeps
    attention weights, by which it can evict(): of each sequence of a batch weigh() counts so many of the last new tokens (0:
    all; None: no weights are kept). Calls are ordered on
    `stream` (default: torch's current stream); where torch works on another one, the caller orders the two.

        kv.begin([0, 3], [1, 512])            # one new token for sequence 0, 512 for sequence 3
        for layer in range(layers):
            q = kv.append(layer, k, v, q)     # [513, heads, dim] each; q comes back rotated
            out = kv.attend(layer, q)
    """

    def __init__(self, layers, q_heads, kv_heads, head_dim, pages, page=64, seqs=64, ctx=262144, fmt=F16, tokens=8192,
                 windows=None, rope=None, stream=None, weigh_last=None):
        import torch
        self._owner = _Handle()
        s = stream if stream is not None else torch.cuda.current_stream()
        self._stream, self.device = s, s.device
        self.layers, self.q_heads, self.kv_heads, self.head_dim = layers, q_heads, kv_heads, head_dim
        self.num_pages, self.page, self.seqs, self.ctx, self.fmt, self.rope = pages, page, seqs, ctx, fmt, rope
        self._config = _config(layers, q_heads, kv_heads, head_dim, pages, page, seqs, ctx, fmt, tokens)
        w, wp = (None, None) if windows is None else _ints([x or 0 for x in windows], layers, "windows")
        with torch.cuda.device(self.device):
            _check(lib().mpg_create(ctypes.byref(self._owner.ptr), ctypes.byref(self._config), wp,
                                    None if rope is None else ctypes.byref(rope.c), ctypes.c_void_p(s.cuda_stream)))
            if weigh_last is not None:
                _check(lib().mpg_keep_weights(self._owner.ptr, _int(weigh_last, "weigh_last")))
        self._h = self._owner.ptr
        self.dtype = _dtype(fmt)
        self._views = {}
        self._lib, self._empty, self._empty_like, self._float32 = lib(), torch.empty, torch.empty_like, torch.float32
        self._scale = head_dim ** -0.5
        self._raw, self._now = s.cuda_stream, torch._C._cuda_getCurrentRawStream  # (a torch stream object costs 2 us a call)

    def close(self):
        """Frees the cache's memory now (tensors that pages() and weights() gave must not be used any more; every call is
        refused from here on); without it, it is freed with the last of the cache and those tensors."""
        self._views.clear()
        self._owner.close()
        self._h = self._owner.ptr

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.close()

    @property
    def handle(self):
        """The handle's mpg_t* (ctypes.c_void_p), for a caller that calls the C ABI through lib() directly."""
        return self._h

    def set_stream(self, stream):
        if stream.device != self.device:
            raise ValueError(f"the stream is on {stream.device}, the cache on {self.device}")
        _check(lib().mpg_set_stream(self._h, ctypes.c_void_p(stream.cuda_stream)))
        self._stream, self._raw = stream, stream.cuda_stream

    def sync(self):
        _check(lib().mpg_sync(self._h))

    # ---- sequences and pages ----

    def length(self, seq):
        n = ctypes.c_int()
        _check(lib().mpg_len(self._h, _int(seq, "sequence"), ctypes.byref(n)))
        return n.value

    def position(self, seq):
        """Where the sequence's next token stands: its length, and the positions evicted of it."""
        n = ctypes.c_int()
        _check(lib().mpg_position(self._h, _int(seq, "sequence"), ctypes.byref(n)))
        return n.value

    def table(self, seq):
        """The sequence's pages, in order."""
        n = _check(lib().mpg_table(self._h, _int(seq, "sequence"), None, 0))
        t = (ctypes.c_int * max(n, 1))()
        _check(lib().mpg_table(self._h, seq, t, n))
        return list(t)[:n]

    def free_pages(self):
        n = ctypes.c_int()
        _check(lib().mpg_free_pages(self._h, ctypes.byref(n)))
        return n.value

    def reserve(self, seqs, counts):
        """Lengthens the sequences by `counts` positions that the caller fills in itself (pages())."""
        (a, ap), (b, bp) = _ints(seqs), _ints(counts, len(seqs), "counts")
        _check(self._lib.mpg_reserve(self._h, len(a), ap, bp))

    def begin(self, seqs, counts, shared=False):
        """Lengthens the sequences by `counts` new tokens and makes them the batch of the appends and attention that
        follow; returns the number of tokens. shared: pages that several of the sequences have in common (forks of one prompt)
        are attended once for all of them, where that is worth it (planning it takes up to 35 us more of the host)."""
        n = ctypes.c_int()
        (a, ap), (b, bp) = _ints(seqs), _ints(counts, len(seqs), "counts")
        call = self._lib.mpg_begin_shared if shared else self._lib.mpg_begin
        _check(call(self._h, len(a), ap, bp, ctypes.byref(n)))
        return n.value

    def set_len(self, seq, n):
        """Shortens a sequence (rollback)."""
        _check(self._lib.mpg_set_len(self._h, _int(seq, "sequence"), _int(n, "length")))

    def fork(self, src, dst, lens=None):
        """Each empty dst[i] becomes the first lens[i] positions of src[i] (all by default); full pages are shared."""
        n = len(dst)
        (a, ap), (b, bp) = _ints(src, n, "src"), _ints(dst)
        c, cp = (None, None) if lens is None else _ints(lens, n, "lens")
        _check(self._lib.mpg_fork(self._h, n, ap, bp, cp))

    def copy(self, src, dst):
        """Each empty dst[i] becomes src[i] on pages of its own."""
        n = len(dst)
        (a, ap), (b, bp) = _ints(src, n, "src"), _ints(dst)
        _check(self._lib.mpg_copy(self._h, n, ap, bp))

    def free(self, seqs):
        a, ap = _ints(seqs)
        _check(self._lib.mpg_free(self._h, len(a), ap))

    def compact(self):
        """Moves pages so that those in use are the lowest; returns how many moved."""
        n = ctypes.c_int()
        _check(self._lib.mpg_compact(self._h, ctypes.byref(n)))
        return n.value

    def evict(self, seqs, keep, first=0, recent=0):
        """Cuts each of the sequences that is longer to `keep` positions (a number, or one for each): its `first` first and
        `recent` last ones and, for each layer and K/V head by itself, those of the largest weights between them. The pool needs
        free pages for all that the call keeps before it gives any back: cut one sequence a call where few are free."""
        a, ap = _ints(seqs)
        b, bp = _ints(keep if hasattr(keep, "__iter__") else [keep] * len(a), len(a), "keep")
        _check(self._lib.mpg_evict(self._h, len(a), ap, bp, _int(first, "first"), _int(recent, "recent")))

    def weights(self, layer):
        """A layer's accumulated attention weights, [sequence, K/V head, position] (f32); those behind a sequence's length are
        undefined."""
        view = self._views.get((layer, "weights"))
        if view is None:
            import torch
            base, by_seq, by_head = ctypes.c_void_p(), ctypes.c_int64(), ctypes.c_int64()
            _check(lib().mpg_weights(self._h, _int(layer, "layer"), ctypes.byref(base), ctypes.byref(by_seq), ctypes.byref(by_head)))

            class _Mem:  # the tensor keeps the memory
                owner = self._owner
                __cuda_array_interface__ = {"shape": (self.seqs, self.kv_heads, self.ctx), "typestr": "<f4", "version": 2,
                                            "strides": (4 * by_seq.value, 4 * by_head.value, 4), "data": (base.value, False)}

            view = self._views[layer, "weights"] = torch.as_tensor(_Mem(), device=self.device)
        return view

    def pages(self, layer, which):
        """A layer's K or V pages as a tensor over the pool: K [page][kv head][pos/16][d/8][16][8], V [page][kv head]
        [pos/32][4][d][8] (element e of group g of V: position 16 (e/4) + 4 g + e%4 of its 32)."""
        view = self._views.get((layer, which))
        if view is None:
            import torch
            base = ctypes.c_void_p()
            _check(lib().mpg_pages(self._h, _int(layer, "layer"), _int(which, "which"), ctypes.byref(base)))
            h, p, d = self.kv_heads, self.page, self.head_dim
            shape = (self.num_pages, h, p // 16, d // 8, 16, 8) if which == K else (self.num_pages, h, p // 32, 4, d, 8)

            class _Mem:  # the tensor keeps the memory
                owner = self._owner
                __cuda_array_interface__ = {"shape": shape, "typestr": "<i2", "data": (base.value, False), "version": 2}

            view = self._views[layer, which] = torch.as_tensor(_Mem(), device=self.device).view(self.dtype)
        return view

    def read_rows(self, layer, which, seq, p0=0, p1=None, out=None):
        """Positions [p0, p1) of a sequence's K or V, [p1 - p0, kv_heads, head_dim]."""
        if p1 is None:
            p1 = self.length(seq)
        n = max(0, p1 - p0)
        if out is None:
            out = self._new((n, self.kv_heads, self.head_dim))
        _rows(out, self.kv_heads, self.head_dim, self.dtype, self.device, "out")
        if out.shape[0] != n or not out.is_contiguous():
            raise ValueError(f"out must be {n} contiguous rows")
        _check(lib().mpg_read_rows(self._h, _int(layer, "layer"), _int(which, "which"), _int(seq, "sequence"),
                                   _int(p0, "position"), _int(p1, "position"), ctypes.c_void_p(out.data_ptr())))
        return out

    # ---- the layers' calls ----

    def _new(self, shape, like=None):
        """An output (like: a tensor of its shape and type). Where torch's current stream is another than the cache's,
        memory that is free on the one may still be in use on the other: it comes from the cache's stream and is held for
        both."""
        if self._now(self.device.index) == self._raw:
            if like is not None and like.is_contiguous():
                return self._empty_like(like)
            return self._empty(shape, dtype=self.dtype, device=self.device)
        import torch
        now = torch.cuda.current_stream(self.device)
        with torch.cuda.stream(self._stream):
            out = self._empty(shape, dtype=self.dtype, device=self.device)
        out.record_stream(now)
        return out

    def _whole(self, t, rows, what):
        """The address of a contiguous [rows, q_heads, head_dim] tensor that takes an output."""
        p = _rows(t, self.q_heads, self.head_dim, self.dtype, self.device, what)[0]
        if t.shape[0] != rows or not t.is_contiguous():
            raise ValueError(f"{what} must be {rows} contiguous rows")
        return p

    def _sinks(self, sinks):
        if sinks.device != self.device or sinks.dtype is not self._float32 or sinks.shape != (self.q_heads,) or not sinks.is_contiguous():
            raise ValueError(f"sinks must be {self.q_heads} contiguous float32 on {self.device}")
        return sinks.data_ptr()

    def append(self, layer, k, v, q=None, q_out=None, rotate=None):
        """Writes the batch's k and v [tokens, kv_heads, head_dim] into the pages, k rotated (rotate=False: it is already;
        default: if the cache has a rope). With q [tokens, q_heads, head_dim]: returns it rotated, in q_out (may be q)."""
        if not -0x80000000 <= layer < 0x80000000:
            _int(layer, "layer")
        rows, h, d = k.shape[0], self.kv_heads, self.head_dim
        kp, kt, kh = _rows(k, h, d, self.dtype, self.device, "k")
        vp, vt, vh = _rows(v, h, d, self.dtype, self.device, "v")
        if v.shape[0] != rows or (q is not None and q.shape[0] != rows):
            raise ValueError("k, v and q differ in rows")
        qp, qt, qh, qo = None, 0, 0, None
        if q is not None:
            qp, qt, qh = _rows(q, self.q_heads, d, self.dtype, self.device, "q")
            if q_out is None:
                q_out = self._new((rows, self.q_heads, d), q)
                qo = q_out.data_ptr()
            else:
                qo = self._whole(q_out, rows, "q_out")
        if rotate is None:
            rotate = self.rope is not None
        rc = self._lib.mpg_append(self._h, layer, rows, kp, kt, kh, vp, vt, vh, qp, qt, qh, qo, 1 if rotate else 0)
        if rc:
            _check(rc)
        return q_out

    def attend(self, layer, q, scale=None, sinks=None, gate=None, out=None):
        """Attention of the batch's tokens: q [tokens, q_heads, head_dim] -> out of the same shape. scale: 1/sqrt(head_dim)
        by default; sinks [q_heads] f32; gate as q: out = attention * sigmoid(gate)."""
        if not -0x80000000 <= layer < 0x80000000:
            _int(layer, "layer")
        h, d, dtype, device = self.q_heads, self.head_dim, self.dtype, self.device
        qp, qt, qh = _rows(q, h, d, dtype, device, "q")
        rows = q.shape[0]
        if out is None:
            out = self._new((rows, h, d), q)
            op = out.data_ptr()
        else:
            op = self._whole(out, rows, "out")
        gp, gt, gh, sp = None, 0, 0, None
        if gate is not None:
            gp, gt, gh = _rows(gate, h, d, dtype, device, "gate")
            if gate.shape[0] != rows:
                raise ValueError("q and gate differ in rows")
        if sinks is not None:
            sp = self._sinks(sinks)
        rc = self._lib.mpg_attend(self._h, layer, rows, qp, qt, qh, self._scale if scale is None else scale, sp, gp, gt, gh, op)
        if rc:
            _check(rc)
        return out

    def weigh(self, layer, q, scale=None, sinks=None, decay=1.0):
        """Adds the attention weights that the batch's counted tokens (weigh_last) give to each position, as attend(layer, q)
        has them, summed over the tokens and the query heads of a K/V head, to `decay` times the position's weight."""
        if not -0x80000000 <= layer < 0x80000000:
            _int(layer, "layer")
        qp, qt, qh = _rows(q, self.q_heads, self.head_dim, self.dtype, self.device, "q")
        sp = None if sinks is None else self._sinks(sinks)
        rc = self._lib.mpg_weigh(self._h, layer, q.shape[0], qp, qt, qh, self._scale if scale is None else scale, sp, decay)
        if rc:
            _check(rc)
