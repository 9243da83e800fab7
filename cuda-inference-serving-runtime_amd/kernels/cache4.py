"""The cache that holds keys and values in 4 bits, and that may keep a bounded number of keys: its kernels' checked entry points,
the rules that pick their forms, and the step metadata they want.

A block of 32 coordinates of one token's key (value) is held as a power of two and 32 codes of 4 bits (0, 0.5, 1, 1.5, 2, 3, 4, 6 and
their negatives times the power; csrc/cache4.h has the layout): 4.25 bits a coordinate, a quarter of the bfloat16 cache, and every
held number is a bfloat16 as it is.  Heads of any even size up to 256, pages of a power of two from 8 tokens on, activations in bfloat16
or float32.

  rope_write    turns queries and keys, writes keys and values into the pages
  attention     softmax attention of a step's rows over the pages (prompt portions and single tokens)
  add_weights   adds every key's attention weight, summed over the rows and heads that see it, to what it had
  evict         keeps of each head's keys the last ones and those with the largest sums
  read          what the pages hold, as bfloat16

`attend` is what a mixer calls.  Launches go to the current stream of the tensors' device.  A Plan's workspace belongs to one launch at a
time: two streams need two plans.
The reference has nothing of this kind (its cache is float32 and keeps every key, runtime/cache.py:9-118).
"""
import ctypes as C
import functools
import math
import operator
import struct
from dataclasses import dataclass
from typing import Optional

import numpy as np
import torch

from . import library, ops
from .ops import BF16, F32, KernelError

UNIT = library.CACHE4
MAX_HEAD = 256
_DT = {torch.bfloat16: BF16, torch.float32: F32}
_entries = {}


def padded(dim):
    """A head's coordinates with the zeros that fill its last block."""
    return -(-dim // 32) * 32


def record_bytes(dim, page_size):
    """Bytes of one head's page, keys and values."""
    return page_size * (padded(dim) + padded(dim) // 16)


def supported(dim, page_size):
    return 0 < dim <= MAX_HEAD and dim % 2 == 0 and page_size >= 8 and page_size & (page_size - 1) == 0


# What an entry point takes: a block of bytes with the stream first, laid out as csrc/cache4.hip and cache4.h say (`cisr_call4_bytes` knows them by
# their place here).  ctypes converts 20 arguments in 1.3 us, a pointer to 20 that are packed in 0.4.
_CALLS = {"cisr_write4": "8P10i", "cisr_read4": "5P6i", "cisr_evict4": "8P12i", "cisr_merge4": "6P6i", "cisr_attn4": "9Pq10if", "cisr_weights4": "8Pq14if"}


def _entry(name):
    found = _entries.get(name)
    if found is None:
        lib, kind = library.load(UNIT), name.split("_d")[0]
        call = struct.Struct(_CALLS[kind] + "0P")                  # (filled up to whole pointers, as the compiler does)
        if lib.cisr_call4_bytes(list(_CALLS).index(kind)) != call.size:
            raise library.KernelLibraryError(f"{name}: its arguments take {call.size} bytes here and others in the library")
        fn = getattr(lib, name)
        fn.argtypes = [C.c_char_p, C.c_char_p][:2 if kind == "cisr_evict4" else 1]
        fn.restype = C.c_int
        found = _entries[name] = (fn, call.pack)
    return found


def _t(t, name, dtype, shape, index, align=1):
    """The address of a contiguous tensor of that type and shape on GPU `index` (on so many bytes).  (Asked eight times a call: what is right costs
    half a microsecond, what is wrong is found out afterwards.)"""
    try:
        if t.dtype is dtype and t.shape == shape and t.is_contiguous() and t.get_device() == index:
            at = t.data_ptr()
            if at % align == 0:
                return at
    except AttributeError:
        pass
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise KernelError(f"{name}: expected a GPU tensor")
    if t.dtype != dtype:
        raise KernelError(f"{name}: dtype {t.dtype}, expected {dtype}")
    if tuple(t.shape) != tuple(shape):
        raise KernelError(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")
    if not t.is_contiguous():
        raise KernelError(f"{name}: tensor must be contiguous")
    if t.get_device() != index:
        raise KernelError(f"{name}: on {t.device}, the others on cuda:{index}")
    raise KernelError(f"{name}: must lie on {align} bytes")


def _addresses(tensors, name, dtype, shape, index):
    """`_t` of every one of the tensors.  (One expression for all that are right: 30 of them in 10 us instead of 15.)"""
    try:
        at = [t.data_ptr() for t in tensors if t.dtype is dtype and t.shape == shape and t.is_contiguous() and t.get_device() == index]
        if len(at) == len(tensors):
            return at
    except AttributeError:
        pass
    return [_t(t, name, dtype, shape, index) for t in tensors]


@functools.lru_cache(maxsize=256)
def _record(heads, kv_heads, dim, page_size):
    """Bytes of a head's page, for sizes that the kernels take."""
    if not supported(dim, page_size):
        raise KernelError(f"cache4: heads of {dim} in pages of {page_size}: an even size up to {MAX_HEAD}, a power of two from 8 on")
    if kv_heads <= 0 or heads <= 0 or heads % kv_heads:
        raise KernelError(f"cache4: {heads} query heads are not a multiple of {kv_heads} key/value heads")
    record = record_bytes(dim, page_size)
    if record >= 1 << 31 or kv_heads * record >= 1 << 32:              # (the kernels' offsets within a page)
        raise KernelError(f"cache4: pages of {page_size} tokens of {kv_heads} heads of {dim} take {kv_heads * record} bytes: fewer than 32 bits can say, and a head's fewer than 31")
    return record


def check_pages(kv_heads, dim, page_size):
    """Refuses pages that the kernels do not take."""
    _record(kv_heads, kv_heads, dim, page_size)


def _gpu_of(t, name, dims):
    """The index of the GPU that tensor `t`, of so many dimensions, is on."""
    if not isinstance(t, torch.Tensor) or t.dim() != dims or not t.is_cuda:
        raise KernelError(f"{name}: expected a GPU tensor of {dims} dimensions")
    return t.get_device()


def _pool(pages, name, dims, what):
    """How many pages a pool of so many dimensions has (page numbers are 32-bit)."""
    shape = pages.shape if isinstance(pages, torch.Tensor) else ()
    if len(shape) != dims:
        raise KernelError(f"{name}: expected a GPU tensor of {dims} dimensions")
    n = shape[-3]
    if not 0 < n < 1 << 31:
        raise KernelError(f"{what}: a pool of {n} pages")
    return n


def _launch(name, index, *args, more=()):
    """Runs an entry point on the current stream of GPU `index`."""
    fn, pack = _entries.get(name) or _entry(name)
    try:
        if ops._raw_stream is not None and ops._current_device is not None and ops._current_device() == index:
            code = fn(pack(ops._raw_stream(index), *args), *more)
        else:
            with torch.cuda.device(index):
                code = fn(pack(ops._stream(), *args), *more)
    except struct.error as e:
        raise KernelError(f"{name}: {e}") from None
    if code:
        raise KernelError(f"{name}: HIP error {code}")


@functools.lru_cache(maxsize=256)
def _of_size(name, dim):
    return f"{name}{padded(dim)}"


def _scale(scale):
    if not 0.0 < scale < math.inf:
        raise KernelError(f"cache4: the score scale must be positive, not {scale}")
    return float(scale)


def _window(window):
    if not window:
        return 0
    window = operator.index(window)
    if not 0 < window < 1 << 30:
        raise KernelError(f"cache4: a window of {window} keys")
    return window


# -- writing and reading ------------------------------------------------------------------------------------------

def rope_write(qkv, positions, slots, cos, sin, pages, q, heads, kv_heads, dim, page_size, interleaved=False):
    """Turns queries and keys of the fused projection rows qkv [T, (heads + 2 kv_heads) dim] by the angles of `positions` int32 [T]
    (cos, sin float [max_pos, rot / 2]; pair i of a head is coordinates (i, i + rot / 2), or with `interleaved` (2 i, 2 i + 1)), puts
    the queries into q [T, heads dim] and holds keys and values in the token slots `slots` int32 [T] of `pages` [n, kv_heads, bytes];
    a slot that is none (-1) is not written, and none may be there twice.  Positions outside the table are taken as the nearest in it.  qkv stays as it is.  What is held is finite: a NaN becomes zero, an infinity the
    largest number held."""
    record = _record(heads, kv_heads, dim, page_size)
    index = _gpu_of(qkv, "qkv", 2)
    dtype, rows = qkv.dtype, qkv.shape[0]
    if dtype not in _DT:
        raise KernelError("qkv: expected rows of bfloat16 or float32")
    n, table = _pool(pages, "pages", 3, "rope_write"), cos.shape
    if len(table) != 2 or not 0 < 2 * table[1] <= dim or table[0] == 0:
        raise KernelError(f"rope_write: angles {tuple(table)} do not fit heads of {dim}")
    if rows:
        _launch("cisr_write4", index, _t(qkv, "qkv", dtype, (rows, (heads + 2 * kv_heads) * dim), index), _t(positions, "positions", torch.int32, (rows,), index),
                _t(slots, "slots", torch.int32, (rows,), index), _t(cos, "cos", torch.float32, table, index), _t(sin, "sin", torch.float32, table, index),
                _t(pages, "pages", torch.uint8, (n, kv_heads, record), index, 16), _t(q, "q", dtype, (rows, heads * dim), index), rows, heads, kv_heads, dim,
                2 * table[1], page_size, n, table[0], int(bool(interleaved)), _DT[dtype])
    return q


def read(storage, slots, keys, values, kv_heads, dim, page_size):
    """What token slots `slots` int32 [T] hold at every site of `storage` [sites, n, kv_heads, bytes]: keys and values bfloat16
    [sites, T, kv_heads, dim], exactly; zeros for a slot that is none."""
    record = _record(kv_heads, kv_heads, dim, page_size)
    index = _gpu_of(storage, "storage", 4)
    n, sites, rows = _pool(storage, "storage", 4, "read"), storage.shape[0], slots.shape[0]
    shape = (sites, rows, kv_heads, dim)
    if rows and sites:
        _launch("cisr_read4", index, _t(storage, "storage", torch.uint8, (sites, n, kv_heads, record), index, 16), _t(slots, "slots", torch.int32, (rows,), index),
                _t(keys, "keys", torch.bfloat16, shape, index, 16), _t(values, "values", torch.bfloat16, shape, index, 16), sites, rows, kv_heads, dim, page_size, n)
    return keys, values


# -- plans ----------------------------------------------------------------------------------------------------------

COMPUTE_UNITS = 256
STEP = 32                  # keys of a step of the kernels
LEAST_PIECE = 16           # steps of a piece of a row's keys, at least: four for each of the four waves that share them


def tile_of(form):
    """Items (a row and a query head of the group that shares a key head) of a block."""
    return (16, 32, 128)[form]


def launch_of(rows, segments, decode_only, heads, kv_heads, dim, dtype):
    """(form, rows of a task) for a step of `rows` rows in `segments` segments.  Forms 0 and 1: a block is 16 or 32 items whose four
    waves share the keys; form 2: four waves of 32 items that walk the keys side by side.
    Microseconds by form, 0 / 1 / 2: 1,024 rows of 9 heads of 64 10 / 14 / 27, 2,048 rows 20 / 19 / 32, 8,192 rows 206 / 158 / 182; 512 rows of 32 heads of 128
    17 / 15 / 24, 1,024 rows 33 / 34 / 46, 1,536 rows 58 / 56 / 59, 2,048 rows 92 / 81 / 77, 4,096 rows 290 / 235 / 196; 4,096 rows of 24 heads of 96
    219 / 184 / 145; 8,192 rows of 16 heads of 64 329 / 250 / 225.  (Small heads change over earlier than the rule says: 4,096 rows of 32 heads of 32 123 / 91 / 83.)"""
    group = heads // kv_heads
    form = 0
    if not decode_only and dtype == torch.bfloat16 and padded(dim) <= 128:
        items = rows * group * kv_heads
        form = 2 if items * padded(dim) >= 96 * 256 * COMPUTE_UNITS else 1 if items >= 32 * 2 * COMPUTE_UNITS else 0
    return form, 1 if decode_only else max(1, tile_of(form) // group)


def pieces_for(kv_heads, group, rows_per_task, form, decode_only):
    """Pieces that all keys of a step are cut into, at least: blocks for four a compute unit, for two where rows of a prompt make many tiles anyway.
    (Two, three, four, six and eight of single tokens: 32 of 16k keys 87, 86, 76, 79, 78 us, 8 of 4k keys 19, 17, 17, 18, 19.  Of prompts one, two, three:
    64 rows behind 8,000 keys 35, 31, 31 us, 3,000 rows behind 3,000 97, 96, 96.)"""
    return max(1, (4 if decode_only else 2) * COMPUTE_UNITS // (kv_heads * -(-rows_per_task * group // tile_of(form))))


def fill_pieces(tasks, merges, counts, cached, rows_per_task, pieces, window, turn=0):
    """Writes the tasks of a step (int32 [n, 8], see csrc/cache4_attention.inc) and its merges ([m, 4]: first row, rows, first piece, pieces; -1: none),
    unused ones at the end; returns how many tasks and merges there are.  Tiles of `rows_per_task` rows of a segment; the keys of long
    ones are cut so that all pieces are about as long as `pieces` of them would be, the longest first; of the second `turn` tasks, which join the
    first on their compute units, the longest last.  (2,048 rows of 9 heads of 64: 21.8 us without that, 20.5 with it; 4,000 rows of 32 heads of
    128: 307, 296.)  Cut is what is half as long again as a piece; where there are as many tiles as pieces anyway, what is two and a half times as long: a prompt's
    last rows have twice the keys of the average, and are better left whole (2,048 rows take 18.5 us, and 26 when the longer ones are cut), but a row behind many
    keys beside them would be walked by one block a head (with 2,048 rows of 32 heads of 128 one row of 32k keys 869 us whole, 84 cut, one of 4k 116 and 73, 64
    rows behind 32k 926 and 117; limits of two and a half to four times do alike, where both cut).  Where the rest of the step hides the longer rows, the merge is
    lost: 250 single rows of 500 keys and six of 4k take 36 us whole and 40 cut."""
    counts, cached = np.asarray(counts, dtype=np.int64), np.asarray(cached, dtype=np.int64)
    tiles = -(-counts // rows_per_task)
    n = int(tiles.sum())
    seg = np.repeat(np.arange(len(counts)), tiles)
    firsts = (np.arange(n) - np.repeat(np.cumsum(tiles) - tiles, tiles)) * rows_per_task
    row0 = (np.cumsum(counts) - counts)[seg] + firsts
    rows = np.minimum(rows_per_task, counts[seg] - firsts)
    sees = cached[seg] + firsts + 1
    first = np.maximum(0, sees - window) // STEP if window else np.zeros(n, dtype=np.int64)
    steps = -(-(sees + rows - 1) // STEP) - first
    each = max(LEAST_PIECE, -(-int(steps.sum()) // pieces))
    cuts = np.where(2 * steps >= (3 if n < pieces else 5) * each, -(-steps // each), 1)
    share = -(-steps // cuts)
    cuts = -(-steps // share)
    of = np.repeat(np.arange(n), cuts)
    number = np.arange(len(of)) - np.repeat(np.cumsum(cuts) - cuts, cuts)
    split = cuts > 1
    piece = np.cumsum(split[of]) - 1
    made = np.stack([seg[of], row0[of], rows[of], sees[of], first[of] + number * share[of], first[of] + np.minimum((number + 1) * share[of], steps[of]),
                     np.where(split[of], piece, -1), np.zeros_like(of)], 1)
    made = made[np.argsort(made[:, 4] - made[:, 5], kind="stable")]
    if turn:
        made[turn:2 * turn] = made[turn:2 * turn][::-1].copy()
    tasks[:len(of)] = made
    tasks[len(of):] = -1
    m = int(split.sum())
    if m:
        begin = np.cumsum(np.where(split, cuts, 0)) - cuts
        merges[:m] = np.stack([row0, rows, begin, cuts], 1)[split]
    merges[m:] = -1
    return len(of), m


def turn_of(kv_heads, group, rows_per_task, form):
    """Tasks whose blocks give every compute unit one."""
    return max(1, COMPUTE_UNITS // (kv_heads * -(-rows_per_task * group // tile_of(form))))


def most_tasks(rows, segments, rows_per_task, pieces):
    """(tasks, tiles) that `rows` rows in `segments` segments make at most."""
    tiles = -(-rows // rows_per_task) + segments
    return 2 * tiles + pieces, tiles


FEW_ITEMS = 64             # of a segment: rows times heads of the group (csrc/cache4_attention.inc has the same number)


def shares_of(rows, many, span, group, kv_heads):
    """Into how many shares the items (a row and a head of the group) of a segment are cut where the keys' attention weights are summed, by the `rows` of
    the longest; 0: every segment has few items, a wave has them all and walks the keys.  Segments of few items beside `many` longer ones are summed that way
    all the same, by a launch of their own: 480 rows and 31 single ones behind 2k keys, 32 heads over 8 of 128, take 298 us together in waves that have
    all items and 38 so, 1,024 rows and 32 single ones behind 8k keys 194 in blocks that share keys and 97, 512 rows and one behind 8k 33 and 38.
    Blocks (128 keys and a share) for three a compute unit, of which two run at once and those of shares that
    no row of is left for leave at once, 256 items a share at least.  (2,048 rows of 9 heads of 64 over 3: 15.6 us with two, 13.5 with three, 16 with four; behind
    2,048 keys 23.4 with two, 24.9 with three; behind 6,144 48 and 43.)"""
    items = rows * group
    if items <= FEW_ITEMS:
        return 0
    blocks = -(-span // 128) * kv_heads * max(1, many)
    return max(1, min(3 * COMPUTE_UNITS // blocks, items // 256, 65535 // max(1, many)))


@dataclass(eq=False)
class Plan:
    """A step as the kernels take it: which rows belong to which segment, how many keys each sees, and the launch shapes."""
    rows: int
    n_segments: int
    span: int                          # keys of the longest segment, rounded up or not
    heads: int
    kv_heads: int
    dim: int
    window: int                        # of the keys that a row sees; 0: all of them
    form: int
    rows_per_task: int
    tasks: torch.Tensor                # int32 [n, 8]
    merges: Optional[torch.Tensor]     # int32 [m, 4], where keys are in several pieces
    pieces: int = 0                    # pieces that leave partial results, at most
    segments: Optional[torch.Tensor] = None      # int32 [S, 5], those of most rows first: first row, rows, keys before the first row, state slot, segment
    slots_below: int = 0               # state slots lie below this number
    shares: int = 0                    # see shares_of
    room: Optional[torch.Tensor] = None          # floats for partial results: of `attention` room_of, of `add_weights` parts_of (one after the other)
    few: bool = False                  # whether a segment has few items
    many: int = 0                      # segments that have more

    def __post_init__(self):
        self.index = self.tasks.get_device()
        if self.room is None and max(self.room_of, self.parts_of):
            self.room = torch.empty(max(self.room_of, self.parts_of), dtype=torch.float32, device=self.tasks.device)
        if self.room is not None and self.room.numel() < max(self.room_of, self.parts_of):
            raise KernelError("cache4: a plan's workspace is too small")

    @property
    def room_of(self):
        return self.pieces * self.rows_per_task * self.heads * (self.dim + 2)

    @property
    def parts_of(self):
        return self.shares * self.many * self.kv_heads * self.span if self.shares > 1 else 0


def _whole(numbers, name, least, n=None):
    out = [operator.index(x) for x in numbers]
    if n is not None and len(out) != n:
        raise KernelError(f"cache4.plan: {len(out)} {name} for {n} segments")
    if any(not least <= x < 1 << 30 for x in out):
        raise KernelError(f"cache4.plan: {name} out of range")
    return out


def plan(counts, cached, heads, kv_heads, dim, window=None, device="cuda:0", state_slots=None, dtype=torch.bfloat16):
    """The Plan of a step: segment s brings counts[s] rows (queries) behind cached[s] keys of its request, whose own keys are in the
    pages too: its row i sees keys 0 .. cached[s] + i (or the last `window` of them).  `state_slots`: where `add_weights` adds a segment's sums,
    each slot once.  `dtype`: the rows' type."""
    if kv_heads <= 0 or heads <= 0 or heads % kv_heads or not supported(dim, 8) or dtype not in _DT:
        raise KernelError(f"cache4.plan: {heads} heads over {kv_heads} of {dim} coordinates in {dtype}")
    counts = _whole(counts, "counts", 1)
    cached = _whole(cached, "cached keys", 0, len(counts))
    window = _window(window)
    if not counts:
        raise KernelError("cache4.plan: a step needs a segment")
    rows, segments = sum(counts), len(counts)
    longest = max(c + n for c, n in zip(cached, counts))
    decode_only = rows == segments
    group = heads // kv_heads
    form, per_task = launch_of(rows, segments, decode_only, heads, kv_heads, dim, dtype)
    return _plan(counts, cached, heads, kv_heads, dim, window, torch.device(device), state_slots, form, per_task,
                 pieces_for(kv_heads, group, per_task, form, decode_only))


def _listed(firsts, counts, cached, slots):
    """int32 [S, 5] of the segments as `add_weights` takes them, those of most rows first."""
    made = np.stack([firsts, counts, cached, slots, np.arange(len(counts))], 1).astype(np.int32)
    return made[np.argsort(-made[:, 1], kind="stable")]


def _plan(counts, cached, heads, kv_heads, dim, window, device, state_slots, form, per_task, pieces):
    rows, segments, group = sum(counts), len(counts), heads // kv_heads
    longest, many = max(c + n for c, n in zip(cached, counts)), sum(c * group > FEW_ITEMS for c in counts)
    tasks, merges = (np.empty((n, k), dtype=np.int32) for n, k in zip(most_tasks(rows, segments, per_task, pieces), (8, 4)))
    n, m = fill_pieces(tasks, merges, counts, cached, per_task, pieces, window, turn_of(kv_heads, group, per_task, form))
    listed = None
    if state_slots is not None:
        slots = _whole(state_slots, "state slots", 0, segments)
        if len(set(slots)) != segments:
            raise KernelError("cache4.plan: two segments with one state slot")
        firsts = np.concatenate(([0], np.cumsum(counts)[:-1]))
        listed = torch.from_numpy(_listed(firsts, counts, cached, slots)).to(device)
    parts = int(tasks[:n, 6].max()) + 1
    return Plan(rows, segments, longest, heads, kv_heads, dim, window, form, per_task, torch.from_numpy(tasks[:n]).to(device),
                torch.from_numpy(merges[:m]).to(device) if m else None, parts, listed, 0 if listed is None else 1 + max(slots),
                0 if listed is None else shares_of(max(counts), many, longest, group, kv_heads), few=many < segments, many=many)


def _planned(plan, q, tables, pages, heads, kv_heads, dim, page_size, window, what):
    """(GPU, bytes of a head's page, pages, the tables' shape) of a planned step, checked against its plan."""
    record = _record(heads, kv_heads, dim, page_size)
    index = _gpu_of(q, "q", 2)
    if not isinstance(plan, Plan) or (plan.heads, plan.kv_heads, plan.dim) != (heads, kv_heads, dim):
        raise KernelError(f"{what}: the plan is of other heads")
    if plan.window != (window or 0):
        raise KernelError(f"{what}: a window of {window} keys, planned: {plan.window}")
    if q.dtype not in _DT or (plan.form > 0 and q.dtype is not torch.bfloat16):
        raise KernelError(f"{what}: rows in {q.dtype}: bfloat16 or float32, as planned")
    if plan.index != index:
        raise KernelError(f"{what}: rows and plan on different GPUs")
    shape = tables.shape
    if len(shape) != 2 or shape[0] < plan.n_segments or not 0 < shape[1] * page_size < 1 << 31:
        raise KernelError(f"tables: shape {tuple(shape)} for {plan.n_segments} segments")
    return index, record, _pool(pages, "pages", 3, what), shape


# -- attention ------------------------------------------------------------------------------------------------------

def attention(q, pages, tables, plan, out, heads, kv_heads, dim, page_size, scale, window=None, stats=None):
    """out [T, heads dim] = softmax(scale q k^T) v of every row over the keys it sees (see `plan`), held in `pages` [n, kv_heads, bytes] of
    the block tables `tables` int32 [S, W].  Keys behind the table's end, and keys in a page that is none, are not seen; a row that sees
    none gets zeros.  `stats` float [T, heads]: gets the scores' log-sum-exp in powers of two (-inf for a row that sees none), as
    `add_weights` takes it.  Rows that the plan does not name are left as they are."""
    index, record, n, table = _planned(plan, q, tables, pages, heads, kv_heads, dim, page_size, window, "attention")
    dtype, rows = q.dtype, plan.rows
    op = _t(out, "out", dtype, (rows, heads * dim), index, 8)
    sp = 0 if stats is None else _t(stats, "stats", torch.float32, (rows, heads), index)
    po = pm = 0
    if plan.pieces:
        po = plan.room.data_ptr()
        pm = po + 4 * plan.pieces * plan.rows_per_task * heads * dim
    dt = _DT[dtype]
    _launch(_of_size("cisr_attn4_d", dim), index, _t(q, "q", dtype, (rows, heads * dim), index, 16), _t(pages, "pages", torch.uint8, (n, kv_heads, record), index, 16),
            _t(tables, "tables", torch.int32, table, index), plan.tasks.data_ptr(), op, sp, po, pm, n, plan.tasks.shape[0], plan.rows_per_task, heads,
            kv_heads, dim, page_size, table[1], plan.window, plan.form, dt, _scale(scale))
    if plan.merges is not None:
        _launch("cisr_merge4", index, po, pm, plan.merges.data_ptr(), op, sp, plan.merges.shape[0], plan.rows_per_task, heads, kv_heads, dim, dt)
    return out


def add_weights(q, stats, pages, tables, plan, weights, heads, kv_heads, dim, page_size, scale, window=None):
    """weights[slot, key head, key] += the key's attention weight, summed over the segment's rows that see it and the query heads
    that share the key head.  `stats`: what `attention` left for the same rows; weights float [slots, kv_heads, capacity], capacity at least the
    keys of the longest segment.  The same bits every time: a key's sum has one writer."""
    index, record, n, table = _planned(plan, q, tables, pages, heads, kv_heads, dim, page_size, window, "add_weights")
    if plan.segments is None:
        raise KernelError("add_weights: the plan names no state slots")
    if _gpu_of(weights, "weights", 3) != index or weights.shape[1] != kv_heads or weights.shape[2] < plan.span or weights.shape[0] < plan.slots_below:
        raise KernelError(f"weights: shape {tuple(weights.shape)} for {kv_heads} heads of {plan.span} keys in {plan.slots_below} slots")
    # Blocks of four waves a segment and key head: as many as reach each a step of keys, and no more than run at once (three a compute unit).
    # 16 rows of 2k keys, 8 key heads: 4, 6, 8, 12 and 17 blocks each (6 is the rule's) take 10.4, 8.7, 11.3, 10.7 and 10.9 us.
    blocks = max(1, min(-(-plan.span // (4 * STEP)), -(-3 * COMPUTE_UNITS // (kv_heads * plan.n_segments)))) if plan.few or not plan.shares else 0
    slots, _, capacity = weights.shape
    _launch(_of_size("cisr_weights4_d", dim), index, _t(q, "q", q.dtype, (plan.rows, heads * dim), index, 16),
            _t(stats, "stats", torch.float32, (plan.rows, heads), index), _t(pages, "pages", torch.uint8, (n, kv_heads, record), index, 16),
            _t(tables, "tables", torch.int32, table, index), plan.segments.data_ptr(), _t(weights, "weights", torch.float32, weights.shape, index),
            plan.room.data_ptr() if plan.parts_of else 0, n, plan.n_segments, plan.many, plan.span, heads, kv_heads, dim, page_size, table[1], plan.window,
            capacity, slots, plan.shares, blocks, _DT[q.dtype], _scale(scale))
    return weights


# -- a bounded number of keys -----------------------------------------------------------------------------------------

def evict(storage, weights, tables, new_tables, lengths, slots, new_slots, kv_heads, dim, page_size, keep, recent, kept):
    """Each head of each request keeps, of its first lengths[r] keys, the last `recent` and of the others those with the largest sums
    of attention weight, `keep` in all (all of them where there are no more); of equal sums the earlier key stays, a NaN counts least.
    The kept keys and values go, in their order, from the pages of `tables` int32 [R, W] to those of `new_tables` int32 [R, W'] (other
    pages, W' page_size at least `keep`) at every site of `storage` [sites, n, kv_heads, bytes]; their sums from weights[site][slots[r]]
    to weights[site][new_slots[r]] (float [n_slots, kv_heads, capacity] a site; it may be the request's own old slot, never another request's, old or new),
    zeros behind them.  Of a request without keys nothing is read or written but its -1 in `kept`.
    kept int32 [sites, R, kv_heads, keep] gets their indices, -1 behind the last.  lengths, slots, new_slots: int32 [R]."""
    record = _record(kv_heads, kv_heads, dim, page_size)
    keep, recent = operator.index(keep), operator.index(recent)
    if not 0 < keep < 1 << 30 or not 0 <= recent <= keep:
        raise KernelError(f"evict: {recent} last keys of {keep}")
    index = _gpu_of(storage, "storage", 4)
    n, sites, requests = _pool(storage, "storage", 4, "evict"), storage.shape[0], lengths.shape[0]
    if len(weights) != sites or sites == 0:
        raise KernelError(f"evict: sums of {len(weights)} sites for {sites}")
    _gpu_of(weights[0], "weights", 3)
    n_slots, _, capacity = weights[0].shape
    if capacity < keep:
        raise KernelError(f"evict: sums of {capacity} keys, {keep} are kept")
    if tables.dim() != 2 or new_tables.dim() != 2 or tables.shape[1] == 0 or new_tables.shape[1] * page_size < keep:
        raise KernelError(f"evict: tables {tuple(tables.shape)} and {tuple(new_tables.shape)} for {keep} keys")
    sums = _addresses(weights, "weights", torch.float32, (n_slots, kv_heads, capacity), index)
    if requests:
        _launch("cisr_evict4", index, _t(lengths, "lengths", torch.int32, (requests,), index), _t(slots, "slots", torch.int32, (requests,), index),
                _t(new_slots, "new_slots", torch.int32, (requests,), index), _t(tables, "tables", torch.int32, (requests, tables.shape[1]), index),
                _t(new_tables, "new_tables", torch.int32, (requests, new_tables.shape[1]), index),
                _t(storage, "storage", torch.uint8, (sites, n, kv_heads, record), index, 16),
                _t(kept, "kept", torch.int32, (sites, requests, kv_heads, keep), index), sites, n, requests, kv_heads, dim, page_size, tables.shape[1],
                new_tables.shape[1], keep, recent, capacity, n_slots, more=(struct.pack(f"{sites}P", *sums),))
    return kept


# -- a step of the engine -----------------------------------------------------------------------------------------------

@dataclass(frozen=True)
class StepForm:
    """Step array without words whose launch value says how a step's rows are taken: 2 to the power of twice the form, and once more where
    keys are in several pieces (powers of two: captured programs round launch values up to them)."""
    pieces: "StepPieces"

    def words(self, rows, segments):
        return 0

    def launch_value(self, batch):
        _, merges, form = self.pieces.made(batch)
        return 1 << (2 * form + (1 if len(merges) else 0))

    def fill(self, out, batch, value):
        pass


@dataclass(frozen=True)
class StepPieces:
    """Step array: the tasks of a step (see fill_pieces), then, from the end backwards, its merges.  Its launch value is the number of tasks."""
    heads: int
    kv_heads: int
    dim: int
    window: int
    half: bool                 # rows in bfloat16

    def launch(self, rows, segments, decode_only):
        """(form, rows of a task, pieces) for a step."""
        form, per_task = launch_of(rows, segments, decode_only, self.heads, self.kv_heads, self.dim, torch.bfloat16 if self.half else torch.float32)
        return form, per_task, pieces_for(self.kv_heads, self.heads // self.kv_heads, per_task, form, decode_only)

    def most(self, rows, segments):
        """(tasks, merges) at most: of a step of single tokens, or of prompts by the smallest tiles."""
        group = self.heads // self.kv_heads
        tasks, tiles = zip(most_tasks(rows, segments, 1, pieces_for(self.kv_heads, group, 1, 0, True)) if rows == segments else (0, 0),
                           most_tasks(rows, segments, max(1, 16 // group), 2 * COMPUTE_UNITS))
        return max(tasks), max(tiles)

    def made(self, batch):
        """(tasks, merges, form) of the batch."""
        got = batch.made.get(self)
        if got is None:
            rows, segments = sum(batch.counts), len(batch.counts)
            form, per_task, pieces = self.launch(batch.rows or rows, segments, batch.decode_only)
            tasks, merges = (np.empty((n, k), dtype=np.int32) for n, k in zip(most_tasks(rows, segments, per_task, pieces), (8, 4)))
            n, m = fill_pieces(tasks, merges, batch.counts, batch.cached, per_task, pieces, self.window,
                               turn_of(self.kv_heads, self.heads // self.kv_heads, per_task, form))
            got = batch.made[self] = (tasks[:n], merges[:m], form)
        return got

    def words(self, rows, segments):
        tasks, merges = self.most(rows, segments)
        return 8 * tasks + 4 * merges

    def launch_value(self, batch):
        return len(self.made(batch)[0])

    def fill(self, out, batch, value):
        tasks, merges, _ = self.made(batch)
        out[:] = -1
        out[:8 * len(tasks)] = tasks.reshape(-1)
        if len(merges):
            out[len(out) - 4 * len(merges):] = merges.reshape(-1)


@dataclass(frozen=True)
class StepSegments:
    """Step array: int32 [S, 5] of first row, rows, keys before the first row, state slot and number of every segment, those of most rows first; no rows pad
    it.  Its launch value is the rows of the longest."""

    def words(self, rows, segments):
        return 5 * segments

    def launch_value(self, batch):
        return max(batch.counts)

    def fill(self, out, batch, value):
        out[:] = 0
        out[:5 * len(batch.counts)] = _listed(batch.first_row, batch.counts, batch.cached, batch.slots).reshape(-1)


@dataclass(frozen=True)
class StepItems:
    """Step array without words whose launch value says how many segments have many items (see shares_of), or with `few` whether one has few."""
    group: int
    few: bool

    def words(self, rows, segments):
        return 0

    def launch_value(self, batch):
        many = sum(c * self.group > FEW_ITEMS for c in batch.counts)
        return int(many < len(batch.counts)) if self.few else many

    def fill(self, out, batch, value):
        pass


def step_arrays(heads, kv_heads, dim, window, operand, sums):
    """What `attend` wants of every step, for a layer whose output projection's weights are `operand` (their type is the rows')."""
    if operand is None:
        return []
    pieces = StepPieces(heads, kv_heads, dim, _window(window), operand.dtype is torch.bfloat16)
    return [pieces, StepForm(pieces)] + ([StepSegments(), StepItems(heads // kv_heads, True), StepItems(heads // kv_heads, False)] if sums else [])


def attend(ctx, q, pages, view, out, heads, kv_heads, dim, scale, window=None, sums=None):
    """`attention` of a step's rows, and with `sums` (float [slots, kv_heads, capacity]) `add_weights`.  `ctx` is the step's context, `view`
    the cache group as the step sees it."""
    array = StepPieces(heads, kv_heads, dim, _window(window), q.dtype is torch.bfloat16)
    words, n_tasks = ctx.step_array(array)
    _, flags = ctx.step_array(StepForm(array))
    form, split = divmod(flags.bit_length() - 1, 2)
    most, merges = array.most(ctx.n_rows, ctx.n_segments)
    per_task = 1 if ctx.decode_only else max(1, tile_of(form) // (heads // kv_heads))
    rows, S = ctx.n_rows, ctx.n_segments
    shares, few, many, span, segments = 0, False, 0, ctx.span_hint, None
    if sums is not None:
        segments, longest = ctx.step_array(StepSegments())
        segments = segments.view(S, 5)
        few, many = (ctx.step_array(StepItems(heads // kv_heads, few))[1] for few in (True, False))
        many = min(many, S)                                            # (under a captured program, rounded up)
        span = min(span, sums.shape[2])
        shares = shares_of(longest, many, span, heads // kv_heads, kv_heads)
    pieces = n_tasks if split else 0
    floats = max(pieces * per_task * heads * (dim + 2), shares * many * kv_heads * span if shares > 1 else 0)
    plan = Plan(rows, S, span, heads, kv_heads, dim, _window(window), form, per_task, words[:8 * min(n_tasks, most)].view(-1, 8), words[len(words) - 4 * merges:].view(-1, 4) if split else None,
                pieces, segments, 0 if sums is None else sums.shape[0], shares, ctx.buffer("cache4.room", (floats,), torch.float32) if floats else None, few > 0, many)
    stats = None if sums is None else ctx.buffer("cache4.stats", (rows, heads), torch.float32)
    attention(q, pages, view.tables, plan, out, heads, kv_heads, dim, view.page_size, scale, window, stats)
    if sums is not None:
        add_weights(q, stats, pages, view.tables, plan, sums, heads, kv_heads, dim, view.page_size, scale, window)
    return out
