"""Paged key-value cache: the operators of csrc/er_kv_*.cu.

The reference keeps one sequence's keys and values in one array
(runtime/qwen_moe.py:90-106) and attends over all of it (:264-291). Here the
keys and values of many sequences lie in pages of a pool, in 16 or 32 bits:

  PagedKV        one layer's pools and page table, the handle of every call
  append         RoPE on new tokens' q and k, k and v into their pages
  attend         attention of query rows over their sequences' pages, split
                 over the length; optionally accumulating each position's weight
  PageBounds, page_bounds, select_pages
                 int8 bounds of every page's keys, and the pages whose bounds
                 score best against a query; attend(pages=, counts=) reads
                 only those
  evict          keeps the positions of greatest accumulated weight

All work is queued on the current stream of the cache's device; nothing
waits on the host. Lengths, positions, tables and lists are read on the
device, so a call captured in a CUDA graph serves whatever they hold at
replay. What is wrong with them (a page id outside the pool, a length
outside the table) is found there too: the rows concerned come back as NaN
(their mass with them, all of it where a length or sequence is bad) or stay
unwritten, and PagedKV.check() raises. attend allocates its workspace from
torch's allocator on that stream unless given one.

Infinities: an infinite or NaN key or value behind a row's length changes
nothing. One that is seen makes the row's results what the formula gives,
infinite or NaN; over an fp32 cache they may be NaN where the formula gives an
infinity. Scores of -inf weigh nothing.
"""

from __future__ import annotations

import ctypes as C
import functools

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}


def _need(t, name: str, dtype, device: torch.device, shape=None, contiguous: bool = True) -> None:
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.device == device and \
            (shape is None or t.shape == shape) and (not contiguous or t.is_contiguous()):
        return
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.device != device:
        got = f"{t.dtype} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
        raise ValueError(f"{name}: expected a {dtype} tensor on {device}, got {got}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")


def _apart(shape, stride) -> bool:
    """Whether no two elements of the strided tensor share a place (each stride passes all that smaller ones reach)."""
    reach = 0
    for step, n in sorted((s, n) for s, n in zip(stride, shape) if n > 1):
        if step <= reach:
            return False
        reach += step * (n - 1)
    return True


def _share(a, b) -> bool:
    """Whether two [seqs, heads, n] tensors may share an element: their extents meet, and they are no two
    layers of one array."""
    (a, b) = sorted((a, b), key=lambda t: t.data_ptr())
    size = a.element_size()
    if not a.numel() or not b.numel():
        return False
    apart = (b.data_ptr() - a.data_ptr()) // size
    if apart > sum((n - 1) * s for n, s in zip(a.shape, a.stride())):
        return False
    shape = [max(m, n) for m, n in zip(a.shape, b.shape)]
    return a.stride() != b.stride() or not _apart((2, *shape), (apart, *a.stride()))


def _meet(apart: int, shape, stride) -> bool:
    """Whether two tensors of this shape and these strides (_apart), the second `apart` elements on, share a
    place: whether the distance is a sum of steps, fewer of each dimension than it has elements."""
    dims = sorted(((s, n) for s, n in zip(stride, shape) if n > 1), reverse=True)

    def steps(left, i):
        if i == len(dims):
            return left == 0
        s, n = dims[i]
        return any(abs(m) < n and steps(left - m * s, i + 1) for m in {left // s, -(-left // s)})

    return steps(apart, 0)


def _weights(t, name: str, cache, rows: int, written: bool) -> None:
    if not isinstance(t, torch.Tensor) or t.dim() != 3 or (t.shape[2] > 1 and t.stride(2) != 1):
        raise ValueError(f"{name}: expected [{rows}, {cache.kv_heads}, n] with contiguous positions")
    _need(t, name, torch.float32, cache.device, (rows, cache.kv_heads, t.shape[2]), contiguous=False)
    if written and not t.is_contiguous() and not _apart(t.shape, t.stride()):
        raise ValueError(f"{name}: strides {t.stride()} make elements share memory")


def _on_device(call):
    """The call with its cache's device as the current one (kernels are launched and memory is allocated there)."""

    @functools.wraps(call)
    def on_device(cache, *args, **kwargs):
        if torch._C._cuda_getDevice() == cache._index:
            return call(cache, *args, **kwargs)
        with torch.cuda.device(cache._index):
            return call(cache, *args, **kwargs)

    return on_device


class PagedKV:
    """One layer's cache. k, v [pages, kv_heads, page_size, head_dim] float32
    or bfloat16 on one CUDA device, with any strides that are alike and leave
    the last dimension contiguous and every slot on 16 bytes (so
    [pages, page_size, kv_heads, head_dim] pools are passed transposed);
    table [seqs, width] int32, rows contiguous: the page of each run of
    page_size positions. head_dim: a multiple of 8, at most 256; kv_heads: at
    most 1024. Sequences may share pages, and k and v memory, as long as no call
    writes to them.

    `status` ([1] int32; a new one unless given) collects what the device
    found wrong (check())."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, status: torch.Tensor | None = None):
        if k.dim() != 4 or k.dtype not in _DTYPES or not k.is_cuda:
            raise ValueError(f"k: expected a [pages, kv_heads, page_size, head_dim] float32 or bfloat16 CUDA tensor, "
                             f"got {tuple(k.shape)} {k.dtype} on {k.device}")
        self.device, self.dtype, self._index = k.device, k.dtype, k.device.index
        _need(v, "v", k.dtype, k.device, k.shape, contiguous=False)
        if k.stride() != v.stride() or k.stride(3) != 1:
            raise ValueError(f"k, v: strides {k.stride()}, {v.stride()} (alike, the last dimension contiguous)")
        _need(table, "table", torch.int32, k.device, contiguous=False)
        if table.dim() != 2 or (table.shape[1] > 1 and table.stride(1) != 1):
            raise ValueError("table: expected [seqs, width] with contiguous rows")
        self.k, self.v, self.table = k, v, table
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self.seqs, self.width = table.shape
        self._apart = _apart(k.shape, k.stride())
        self._two = self._apart and not _meet((v.data_ptr() - k.data_ptr()) // k.element_size(), k.shape, k.stride())
        if status is not None:
            _need(status, "status", torch.int32, k.device, (1,))
        self.status = torch.zeros(1, dtype=torch.int32, device=k.device) if status is None else status
        self._status = self.status.data_ptr()
        self._c = _lib.KvCache(
            k=k.data_ptr(), v=v.data_ptr(), dtype=_DTYPES[k.dtype], num_pages=self.num_pages,
            page_size=self.page_size, kv_heads=self.kv_heads, head_dim=self.head_dim, page_stride=k.stride(0),
            head_stride=k.stride(1), slot_stride=k.stride(2), table=table.data_ptr(), seqs=self.seqs,
            table_width=self.width, table_stride=table.stride(0))
        self._ref = C.byref(self._c)
        self._needs: dict[tuple, int] = {}  # workspace bytes by the sizes of a call

    def _stream(self) -> int:
        # the handle of torch.cuda.current_stream(device), without building a Stream object for it
        return torch._C._cuda_getCurrentRawStream(self._index)

    def _writable(self) -> None:
        if not self._apart:
            raise ValueError(f"pools of strides {self.k.stride()} make slots share memory")
        if not self._two:
            raise ValueError("k and v share memory")

    def check(self) -> None:
        """Raises ValueError if a call since the last check met a bad page id,
        length or sequence on the device. Waits for the stream's work."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            what = [t for b, t in ((_lib.KV_BAD_PAGE, "a page id outside the pool"),
                                   (_lib.KV_BAD_LENGTH, "a length, position or count outside its table"),
                                   (_lib.KV_BAD_SEQ, "a sequence outside the table")) if bits & b]
            raise ValueError("paged cache: " + ", ".join(what))


class PageBounds:
    """Per page and key head, the least and greatest key of every channel,
    rounded to the nearest code (a key may pass them by half a step):
    codes [pages, kv_heads, 2, head_dim] int8 and scales [pages, kv_heads]
    float32, contiguous, on the cache's device."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dim() != 4 or codes.shape[2] != 2:
            raise ValueError(f"codes: expected [pages, kv_heads, 2, head_dim], got {tuple(codes.shape)}")
        _need(codes, "codes", torch.int8, codes.device)
        _need(scales, "scales", torch.float32, codes.device, codes.shape[:2])
        self.codes, self.scales = codes, scales
        self._codes, self._scales = codes.data_ptr(), scales.data_ptr()

    @classmethod
    def new(cls, cache: PagedKV) -> PageBounds:
        shape = (cache.num_pages, cache.kv_heads, 2, cache.head_dim)
        return cls(torch.zeros(shape, dtype=torch.int8, device=cache.device),
                   torch.zeros(shape[:2], dtype=torch.float32, device=cache.device))

    def _fit(self, cache: PagedKV) -> None:
        if self.codes.device != cache.device or \
                tuple(self.codes.shape) != (cache.num_pages, cache.kv_heads, 2, cache.head_dim):
            raise ValueError(f"bounds {tuple(self.codes.shape)} on {self.codes.device} are not this cache's")


def _queries(cache: PagedKV, q: torch.Tensor):
    """(rows, heads, row stride) of q [rows, heads, head_dim]."""
    shape = q.shape
    if len(shape) != 3 or shape[2] != cache.head_dim or q.dtype not in _DTYPES or q.device != cache.device:
        raise ValueError(f"q: expected [rows, heads, {cache.head_dim}] float32 or bfloat16 on {cache.device}, "
                         f"got {tuple(shape)} {q.dtype} on {q.device}")
    rows, heads, d = shape
    if heads == 0 or heads % cache.kv_heads:
        raise ValueError(f"q: {heads} heads over {cache.kv_heads} key heads")
    by = q.stride()
    if by[2] != 1 or (heads > 1 and by[1] != d) or (rows > 1 and by[0] < heads * d):
        raise ValueError(f"q: strides {by} (heads contiguous, rows apart)")
    return rows, heads, by[0] if rows > 1 else heads * d


def _row_args(cache: PagedKV, rows: int, lens: torch.Tensor, seqs: torch.Tensor | None, name: str = "lens") -> None:
    _need(lens, name, torch.int32, cache.device, (rows,))
    if seqs is not None:
        _need(seqs, "seqs", torch.int32, cache.device, (rows,))
    elif rows > cache.seqs:
        raise ValueError(f"{rows} rows over {cache.seqs} sequences: give seqs")


def _scratch(need: int, workspace: torch.Tensor | None, device: torch.device) -> torch.Tensor:
    if workspace is None:
        return torch.empty(need, dtype=torch.uint8, device=device)
    if workspace.device != device or not workspace.is_contiguous() or \
            workspace.numel() * workspace.element_size() < need:
        raise ValueError(f"workspace: {need} contiguous bytes on {device} needed")
    if workspace.data_ptr() % 256:
        raise ValueError("workspace: must be 256-byte aligned")
    return workspace


@_on_device
def append(cache: PagedKV, qkv: torch.Tensor, positions: torch.Tensor, heads: int, theta: float, *,
           seqs: torch.Tensor | None = None, slots: torch.Tensor | None = None,
           q_dtype: torch.dtype | None = None) -> torch.Tensor:
    """New tokens into the cache: row i of qkv [n, (heads + 2 kv_heads) head_dim]
    (float32 or bfloat16, rows may be strided) is token positions[i] of
    sequence seqs[i] (default: i) and goes to place slots[i] of it in the
    cache (default: positions[i]; they differ once positions were evicted).
    Returns the queries, rotated, [n, heads, head_dim] in q_dtype (default:
    qkv's); k (rotated) and v go to the pages. A (sequence, place) pair may
    occur once in a call."""
    row = (heads + 2 * cache.kv_heads) * cache.head_dim
    if len(qkv.shape) != 2 or qkv.dtype not in _DTYPES or qkv.device != cache.device or qkv.shape[1] != row or \
            qkv.stride(1) != 1:
        raise ValueError(f"qkv: expected [n, {row}] float32 or bfloat16 on {cache.device}, "
                         f"got {tuple(qkv.shape)} {qkv.dtype} on {qkv.device}")
    n = qkv.shape[0]
    _row_args(cache, n, positions, seqs, "positions")
    if slots is not None:
        _need(slots, "slots", torch.int32, cache.device, (n,))
    cache._writable()
    dt = qkv.dtype if q_dtype is None else q_dtype
    if dt not in _DTYPES:
        raise ValueError(f"q_dtype: float32 or bfloat16, got {dt}")
    q = qkv.new_empty((n, heads, cache.head_dim), dtype=dt)
    _lib.check(_lib.lib().er_kv_append(cache._ref, qkv.data_ptr(), _DTYPES[qkv.dtype],
                                       qkv.stride(0) if n > 1 else row,
                                       None if seqs is None else seqs.data_ptr(), positions.data_ptr(),
                                       None if slots is None else slots.data_ptr(), n, int(heads), float(theta),
                                       q.data_ptr(), _DTYPES[dt], cache._status, cache._stream()), "er_kv_append")
    return q


@_on_device
def attend(cache: PagedKV, q: torch.Tensor, lens: torch.Tensor, *, seqs: torch.Tensor | None = None,
           scale: float | None = None, mass: torch.Tensor | None = None, pages: torch.Tensor | None = None,
           counts: torch.Tensor | None = None, out: torch.Tensor | None = None,
           workspace: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v for rows of queries q [rows, heads, head_dim]
    (float32 or bfloat16; heads a multiple of kv_heads), row r over the first
    lens[r] positions of sequence seqs[r] (default: r). Sums and the softmax
    are in 32 bits; the result has q's dtype and is zero for rows without
    keys. scale: default head_dim ** -0.5.

    mass [rows, kv_heads, n] float32 (the last dimension contiguous): grows
    by each position's attention weight, summed over its key head's queries.
    pages [rows, kv_heads, m], counts [rows, kv_heads] int32 (select_pages):
    only those pages are read, each of them listed once. workspace: scratch of
    one's own instead of a new one (ValueError names the bytes needed); it
    serves one call at a time, captured ones included."""
    rows, heads, stride = _queries(cache, q)
    _row_args(cache, rows, lens, seqs)
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(q.shape)
    else:
        _need(out, "out", q.dtype, cache.device, (rows, heads, cache.head_dim))
    io = _lib.KvAttendIO(
        q=q.data_ptr(), q_dtype=_DTYPES[q.dtype], q_stride=stride, out=out.data_ptr(), rows=rows, heads=heads,
        seqs=None if seqs is None else seqs.data_ptr(), lens=lens.data_ptr(),
        scale=cache.head_dim ** -0.5 if scale is None else float(scale), status=cache._status)
    if (pages is None) != (counts is None):
        raise ValueError("pages and counts go together")
    if pages is not None:
        if mass is not None:
            raise ValueError("mass is not accumulated over page lists")
        if pages.dim() != 3 or pages.shape[2] == 0:
            raise ValueError(f"pages: expected [rows, kv_heads, m], got {tuple(pages.shape)}")
        _need(pages, "pages", torch.int32, cache.device, (rows, cache.kv_heads, pages.shape[2]))
        _need(counts, "counts", torch.int32, cache.device, (rows, cache.kv_heads))
        io.pages, io.counts, io.max_pages = pages.data_ptr(), counts.data_ptr(), pages.shape[2]
    if mass is not None:
        _weights(mass, "mass", cache, rows, True)
        io.mass, io.mass_len = mass.data_ptr(), mass.shape[2]
        io.mass_row_stride, io.mass_head_stride = mass.stride(0), mass.stride(1)
    if rows == 0:
        return out
    lib, ref = _lib.lib(), C.byref(io)
    sizes = (rows, heads, q.dtype, io.max_pages, io.mass_len if mass is not None else -1)
    need = cache._needs.get(sizes)
    if need is None:
        need = cache._needs[sizes] = lib.er_kv_attend_workspace_bytes(cache._ref, ref)
    ws = _scratch(need, workspace, cache.device) if need else None
    _lib.check(lib.er_kv_attend(cache._ref, ref, ws.data_ptr() if need else None, need, cache._stream()),
               "er_kv_attend")
    return out


@_on_device
def page_bounds(cache: PagedKV, bounds: PageBounds, lens: torch.Tensor, start: torch.Tensor) -> None:
    """Renews the bounds of the pages that hold positions [start[s], lens[s])
    of every sequence s, from the page's keys up to lens[s]."""
    bounds._fit(cache)
    _need(lens, "lens", torch.int32, cache.device, (cache.seqs,))
    _need(start, "start", torch.int32, cache.device, (cache.seqs,))
    _lib.check(_lib.lib().er_kv_page_bounds(cache._ref, lens.data_ptr(), start.data_ptr(),
                                            bounds._codes, bounds._scales,
                                            cache._status, cache._stream()), "er_kv_page_bounds")


@_on_device
def select_pages(cache: PagedKV, bounds: PageBounds, q: torch.Tensor, lens: torch.Tensor, budget: int, *,
                 sinks: int = 1, recent: int = 1,
                 seqs: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """For each row and key head up to `budget` pages: the first `sinks`, the
    last `recent`, then those whose bounds allow the greatest product with
    one of the key head's queries. Both enter as int8 codes, rounded to the
    nearest: the choice is exact in them and the same everywhere (ties to the
    lower page), and goes by the keys' true bounds up to half a step of either
    code, a step being a 127th of the greatest value. Returns pages
    [rows, kv_heads, budget] int32, page ordinals ascending with -1 behind
    them, and counts [rows, kv_heads] int32."""
    bounds._fit(cache)
    rows, heads, stride = _queries(cache, q)
    _row_args(cache, rows, lens, seqs)
    if budget <= 0 or sinks < 0 or recent < 0 or sinks + recent > budget:
        raise ValueError(f"budget {budget} with {sinks} first and {recent} last pages")
    lib = _lib.lib()
    pages, counts = lens.new_empty((rows, cache.kv_heads, budget)), lens.new_empty((rows, cache.kv_heads))
    _lib.check(lib.er_kv_select(cache._ref, q.data_ptr(), _DTYPES[q.dtype], stride, rows, heads,
                                None if seqs is None else seqs.data_ptr(), lens.data_ptr(),
                                bounds._codes, bounds._scales, int(budget), int(sinks), int(recent),
                                pages.data_ptr(), counts.data_ptr(), cache._status, cache._stream()), "er_kv_select")
    return pages, counts


@_on_device
def evict(cache: PagedKV, lens: torch.Tensor, mass: torch.Tensor, to: PagedKV, to_mass: torch.Tensor, budget: int, *,
          sinks: int = 4, recent: int = 128) -> tuple[torch.Tensor, torch.Tensor]:
    """Keeps min(lens[s], budget) positions of every sequence and key head:
    the first `sinks`, the last `recent`, then those of the greatest mass
    [seqs, kv_heads, n] (ties to the lower position). They are copied in
    order to positions 0, 1, ... of `to`, whose pages must be none of the
    cache's own that its tables name, and their mass to to_mass; what lies
    behind them stays as it was. Returns kept [seqs, kv_heads, budget] int32
    (-1 behind the last) and the new lengths [seqs] int32."""
    if to.device != cache.device or to.dtype != cache.dtype or to.kv_heads != cache.kv_heads or \
            to.head_dim != cache.head_dim or to.seqs != cache.seqs:
        raise ValueError("to: not a cache of the same device, dtype, key heads, head_dim and sequences")
    if to.table.data_ptr() == cache.table.data_ptr() and to.k.data_ptr() == cache.k.data_ptr():
        raise ValueError("to: the cache's own pages")
    _need(lens, "lens", torch.int32, cache.device, (cache.seqs,))
    _weights(mass, "mass", cache, cache.seqs, False)
    _weights(to_mass, "to_mass", cache, cache.seqs, True)
    to._writable()
    if _share(mass, to_mass):
        raise ValueError("to_mass: must not share memory with mass")
    if budget <= 0 or sinks < 0 or recent < 0 or sinks + recent > budget:
        raise ValueError(f"budget {budget} with {sinks} first and {recent} last positions")
    kept, new = lens.new_empty((cache.seqs, cache.kv_heads, budget)), lens.new_empty(cache.seqs)
    _lib.check(_lib.lib().er_kv_evict(cache._ref, to._ref, lens.data_ptr(), mass.data_ptr(), mass.stride(0),
                                      mass.stride(1), mass.shape[2], to_mass.data_ptr(), to_mass.stride(0),
                                      to_mass.stride(1), to_mass.shape[2], int(budget), int(sinks), int(recent),
                                      kept.data_ptr(), new.data_ptr(), cache._status, cache._stream()),
               "er_kv_evict")
    return kept, new
