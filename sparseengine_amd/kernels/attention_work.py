"""Work list of the matrix-core attention kernels (host side, numpy).

For one step and one (query heads per kv head) ratio: the rows of every item are cut into tiles
of 16.  A step with enough tiles to fill the chip (prompt portions) goes to the kernel that shares
keys and values through shared memory: a unit is a run of ``TILES_PER_BLOCK`` tiles of one item.
A step with few tiles (decoding) goes to the kernel with one wavefront per unit: every tile's keys
are cut into equal ranges (multiples of 32 keys) and a merge task per tile combines them.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import numpy as np

UNIT_FIELDS = 8      # item, row_tile, key_begin, key_end, partial_slot (-1: none), q_start, q_len, ctx_len
TASK_FIELDS = 6      # item, row_tile, first_slot, num_splits, q_start, q_len
# a block's record: item, first_tile, key_begin, key_end, partial_slot of its first tile (-1: none), q_start,
# q_len, ctx_len, slots between two of its tiles (= key ranges per tile), 3 unused
BLOCK_UNIT_FIELDS = 12
# Measured on MI355X (48:8 heads of 128, pages of 64): one wavefront per SIMD is the sweet spot.
# 8 requests x 2048 keys take 20 us in 16 ranges of 128 keys against 24 us in 32 of 64; 64 requests
# x 2060 keys 102 us in 2 ranges (1024 wavefronts) against 146 us unsplit and 118 us in 4 ranges;
# 64 x 8192 keys 360 us (6.0 TB/s) against 550 us unsplit; 4 x 131072 keys 361 us (5.9 TB/s).
TARGET_WAVES = 1024    # wavefronts wanted in flight (256 CUs x 4 SIMDs)
MIN_SPLIT_KEYS = 128   # keys of a range; 64 when ranges of 128 would leave most of the chip idle (one request)
MAX_SPLITS = 256       # what the merge kernel's shared memory holds
TILES_PER_BLOCK = 8    # row tiles of one block of the shared-memory kernel
TILED_MAX_HEAD_DIM = 128
# Blocks, measured the same way (one request, causal flops): a portion of 512 tokens at context 16384 takes
# 322 us in 3 ranges (576 blocks: one round of the chip's 512 places and an eighth of another) and 249 us in 8
# ranges of 2048 keys (three rounds); at context 32768 594 against 443 us, a portion of 2048 at context 8192
# 419 against 393 us.  Ranges under about a thousand keys lose it again to their own start-up and to the merge
# (512 tokens at context 4096: 93 us in 3 or 4 ranges, 99 us in 8), and the rows of a whole prompt see more and
# more keys, so equal ranges leave most of its blocks with half-empty ones (2048 tokens: 75 us whole, 105 us in
# two ranges; 2048 at context 4096: 177 against 218 us): an item's keys are cut up only if the keys before its
# portion are at least three times the portion.
TARGET_BLOCKS = 1536   # blocks wanted in flight (three rounds of two per CU); fewer: their keys are split
MIN_BLOCK_KEYS = 2048
PREFIX_PER_PORTION = 3
WHOLE = 1 << 30        # more keys than any context: not cut into ranges


@dataclass
class AttentionWork:
    """Both lists may be non-empty: a step's prompt portions go to the block kernel, its single
    tokens (whose few rows would leave a block mostly idle over a whole context) to the other."""
    units: np.ndarray        # int32 [num_units, UNIT_FIELDS]: (tile, key range) for one wavefront each
    tasks: np.ndarray        # int32 [num_tasks, TASK_FIELDS]: merges of split tiles
    num_slots: int           # partial results the units write
    block_units: np.ndarray  # int32 [num_block_units, UNIT_FIELDS]: runs of TILES_PER_BLOCK tiles for a block
    tiles_per_block: int = TILES_PER_BLOCK


@dataclass
class DeviceAttentionWork:
    """An ``AttentionWork`` whose lists lie in device memory (int32 tensors)."""
    units: object
    num_units: int
    tasks: object
    num_tasks: int
    num_slots: int
    block_units: object
    num_block_units: int
    tiles_per_block: int


@dataclass
class StepLengths:
    """The lengths that a step's kept work lists are for (under ``"lengths"`` among them)."""
    q_len: object            # ``lengths_key`` of the items' new tokens
    ctx_len: object          # and of their contexts
    numbers: bytes           # both, whatever kind of sequence they came in
    tokens: int              # of the step
    items: int
    longest: int             # context


def lengths_key(lengths):
    """What two equal sequences of lengths of one kind have in common."""
    return lengths.tobytes() if type(lengths) is np.ndarray else tuple(lengths)


def step_lengths(q_len, ctx_len) -> StepLengths:
    both = np.asarray([q_len, ctx_len], dtype=np.int64)
    return StepLengths(lengths_key(q_len), lengths_key(ctx_len), both.tobytes(), int(both[0].sum()), both.shape[1], int(both[1].max()))


# A cache in 4 bits (the same heads; the kernel alone would be bound by reading at one wavefront per SIMD, and a few
# too many, which run beside the others on some SIMDs, cost as much as twice as many everywhere).  4 requests of up to
# 131071 keys take 75 us in at most 1024 ranges, 79 us in 2048; one 34 against 39 us; 8 x 30000 keys 43 against 45; but 64
# requests x 8 heads are 512 tiles, whose ranges come in halves: 64 x 8200 keys 150 us unsplit, 92 us in 1536 ranges.  (The
# numbers of ranges that come of this are not always good ones: 32 x 30000 keys make 768, which leave a quarter of the SIMDs
# idle, 64 x 30000 make 1536, two on one half of the SIMDs and one on the other, 4.6 TB/s where the four requests reach 5.8.)
# A request of 77 keys takes 5.7 us whole and 7.4 in two ranges, 300 keys 9.5 us whole and 8.1 in five.
# At head size 64 a step has half the bytes and one wavefront per SIMD is not enough (4 x 131071 keys, 32:8 heads: 50 us
# in 1024 ranges, 43 in 2048).
FP4_WAVES = 1024            # ranges wanted at head sizes from 128 on, while there are at least four to a tile;
FP4_MANY_WAVES = 2048       # else
FP4_MIN_SPLIT_KEYS = 128
FP4_WHOLE_KEYS = 160        # a step none of whose contexts is longer is not split at all
# Where the tiles alone fill the chip, a range holds at most so many times the mean keys of a tile: 200 requests of 500 keys
# and one of 131071 take 92 us instead of 2302 us, in which one wavefront per kv head goes through all of the long one; 300 of
# 2000 and the same one 201 instead of 2369 us; 200 of 3000 and four of 12000 177 instead of 274 us.  Lengths within twice
# their mean, the ordinary step, are not cut (160 of 4000 to 8200: 273 us).
FP4_MOST_MEANS = 2
# Items in blocks read unpacked pages, which takes a launch and writes and reads four times the bytes, but then every
# product costs less than half: 5.6 against about 2.5 us a row tile and 32768 keys (48:8 heads of 128, one request).  64,
# 128 and 192 rows at 4096 keys take 51, 54 and 57 us in blocks, 32, 49 and 65 directly; 32 and 128 at 32768 keys 80 and 175
# against 81 and 263; 512 at 16384 233 against 528; 32:8 heads of 64: 128 and 256 rows at 4096 keys 38 and 41 against 27
# and 45, 96 at 32768 keys 66 against 87.  An item with at least so many tiles goes in blocks if
# the step's items together have so many tiles beyond that, times the keys they read.
FP4_BLOCK_TILES = 8
FP4_BLOCK_WORK = 196608

_native = None      # the compiled builder (csrc/host_work.hip)


def _native_library():
    """The compiled builder; like every other library of the kernels it is built at first use and
    a failure to build or load it is an error (``KernelLibraryError``), not a quiet change of path."""
    global _native
    if _native is None:
        from . import library
        lib = library.load("host_work")
        i64p, i32p = ctypes.POINTER(ctypes.c_int64), ctypes.POINTER(ctypes.c_int32)
        lib.se_attention_work_plan.argtypes = [i64p, i64p, ctypes.c_int, ctypes.c_int, ctypes.c_int,
                                               ctypes.c_int, ctypes.c_int, i64p, i64p, i64p, i64p]
        lib.se_attention_work_fill.argtypes = [i64p, i64p, ctypes.c_int, ctypes.c_int, ctypes.c_int, i64p,
                                               i64p, i32p, i32p, i32p]
        _native = lib
    return _native


_BAD_LENGTHS = "attention work: every item needs at least one new token and no more new tokens than its context holds"


def build_attention_work(q_len, ctx_len, group: int, kv_heads: int, window: int = 0,
                         target_waves: int = TARGET_WAVES, head_dim: int = 0,
                         min_split_keys: int = MIN_SPLIT_KEYS, block_tiles=TILES_PER_BLOCK // 2,
                         most_keys: int = WHOLE) -> AttentionWork:
    """The work lists of one step, from the compiled builder; ``build_attention_work_numpy`` states
    the rules and gives the same lists (the tests compare the two), about twenty times slower."""
    lib = _native_library()
    q = np.ascontiguousarray(q_len, dtype=np.int64)
    c = np.ascontiguousarray(ctx_len, dtype=np.int64)
    rules = np.asarray([target_waves, min_split_keys, MAX_SPLITS, TILES_PER_BLOCK, TILED_MAX_HEAD_DIM,
                        TARGET_BLOCKS, MIN_BLOCK_KEYS, PREFIX_PER_PORTION, most_keys], dtype=np.int64)
    needed = np.full(q.size, block_tiles, dtype=np.int64)      # a number for all items, or one for each
    plan = np.empty((q.size, 6), dtype=np.int64)
    counts = np.empty(4, dtype=np.int64)
    i64p, i32p = ctypes.POINTER(ctypes.c_int64), ctypes.POINTER(ctypes.c_int32)
    as64 = lambda a: a.ctypes.data_as(i64p)
    status = lib.se_attention_work_plan(as64(q), as64(c), q.size, group, kv_heads, int(window or 0), int(head_dim or 0),
                                        as64(needed), as64(rules), as64(plan), as64(counts))
    if status == -2:
        raise ValueError(_BAD_LENGTHS)
    if status != 0:
        raise ValueError("attention work: bad arguments")
    units = np.empty((int(counts[0]), UNIT_FIELDS), dtype=np.int32)
    tasks = np.empty((int(counts[1]), TASK_FIELDS), dtype=np.int32)
    blocks = np.empty((int(counts[2]), BLOCK_UNIT_FIELDS), dtype=np.int32)
    lib.se_attention_work_fill(as64(q), as64(c), q.size, group, int(window or 0), as64(rules), as64(plan),
                               units.ctypes.data_as(i32p), tasks.ctypes.data_as(i32p), blocks.ctypes.data_as(i32p))
    return AttentionWork(units, tasks, int(counts[3]), blocks)


def build_fp4_attention_work(q_len, ctx_len, group: int, kv_heads: int, window: int = 0, head_dim: int = 0, page: int = 1,
                             most_unpacked: int | None = None) -> AttentionWork:
    """The work lists of a step over a cache in 4 bits: ranges that together are no more than fill the chip once (an
    item's last range is a partial one, so one is taken off the number wanted for each tile)."""
    q = np.asarray(q_len, dtype=np.int64)
    block_tiles = fp4_block_tiles(q, ctx_len, group, window, page, most_unpacked)
    alone = np.where(items_in_blocks(q, group, head_dim, block_tiles), 0, (q * group + 15) // 16)
    tiles = int(alone.sum()) * kv_heads
    wanted = FP4_WAVES if head_dim >= 128 and 4 * tiles <= FP4_WAVES else FP4_MANY_WAVES
    if q.size and int(np.max(ctx_len)) <= FP4_WHOLE_KEYS:
        wanted = 0
    most = WHOLE
    if tiles >= wanted - tiles and tiles:      # no ranges are wanted: an item far above the others gets some all the same
        c = np.asarray(ctx_len, dtype=np.int64)
        mean = -(-int((alone * (np.minimum(c, window + q) if window else c)).sum()) * kv_heads // tiles)
        most = max(FP4_WHOLE_KEYS, -(-FP4_MOST_MEANS * mean // 32) * 32)
    return build_attention_work(q_len, ctx_len, group, kv_heads, window, max(1, wanted - tiles), head_dim, FP4_MIN_SPLIT_KEYS,
                                block_tiles, most)


def fp4_block_tiles(q_len, ctx_len, group: int, window: int, page: int = 1, most_unpacked: int | None = None):
    """The tiles an item needs to go in blocks in a step over a cache in 4 bits: a number, or one for each item where not
    all that have enough may.  ``most_unpacked``: the tokens that the step may unpack, in whole pages of ``page`` (None: no
    limit); those whose rows read the most keys come first, the others stay with the kernel that reads 4 bits."""
    q, c = np.asarray(q_len, dtype=np.int64), np.asarray(ctx_len, dtype=np.int64)
    beyond = np.maximum((q * group + 15) // 16 - FP4_BLOCK_TILES, 0)
    if not beyond.any():
        return FP4_BLOCK_TILES + 1
    reach = np.minimum(c, window + q) if window else c
    if int((beyond * reach).sum()) < FP4_BLOCK_WORK:
        return 1 << 30
    if most_unpacked is None:
        return FP4_BLOCK_TILES
    first, until = _pages_read(q, c, window, page)
    tokens = np.where((q * group + 15) // 16 >= FP4_BLOCK_TILES, (until - first) * page, 0)
    if int(tokens.sum()) <= most_unpacked:
        return FP4_BLOCK_TILES
    needed, left = np.full(q.size, 1 << 30, dtype=np.int64), most_unpacked
    for i in np.argsort(-beyond * reach, kind="stable").tolist():
        if tokens[i] <= left:
            needed[i] = FP4_BLOCK_TILES
            left -= int(tokens[i])
    return needed


def _pages_read(q_len, ctx_len, window: int, page: int):
    """Per item the block-table columns [first, until) that its rows read."""
    low = np.maximum(0, ctx_len - q_len - window + 1) if window else np.zeros_like(ctx_len)
    return low // page, -(-ctx_len // page)


FP4_HEAD_DIMS = (64, 128, 256)      # head sizes that the 4-bit attention kernel is built for


def fp4_unpack_list(q_len, ctx_len, group: int, head_dim: int, page: int, window: int, only_blocks: bool,
                    most_unpacked: int | None = None):
    """Which pages of a 4-bit cache a step reads through unpacked copies (those of the block kernel's items, or of all):
    int32 ``[n, 2]`` (item, column of the block table), and int32 ``[items, columns]`` where each lies among them."""
    q_len, ctx_len = np.asarray(q_len, dtype=np.int64), np.asarray(ctx_len, dtype=np.int64)
    chosen = (items_in_blocks(q_len, group, head_dim, fp4_block_tiles(q_len, ctx_len, group, window, page, most_unpacked))
              if only_blocks else np.ones(q_len.size, dtype=bool))
    first, until = _pages_read(q_len, ctx_len, window, page)
    column = np.arange(int(until.max()))[None, :]
    read = (column >= first[:, None]) & (column < until[:, None]) & chosen[:, None]
    pairs = np.ascontiguousarray(np.argwhere(read), dtype=np.int32)
    table = np.zeros(read.shape, dtype=np.int32)
    table[read] = np.arange(pairs.shape[0], dtype=np.int32)
    return pairs, table


def items_in_blocks(q_len, group: int, head_dim: int, block_tiles=TILES_PER_BLOCK // 2) -> np.ndarray:
    """Which items go to the block kernel: those with at least half a block of tiles, or ``block_tiles`` (a number, or one
    for each item)."""
    tiles = (np.asarray(q_len, dtype=np.int64) * group + 15) // 16
    if not head_dim or head_dim % 32 or head_dim > TILED_MAX_HEAD_DIM:
        return np.zeros(tiles.size, dtype=bool)
    return tiles >= block_tiles


def build_attention_work_numpy(q_len, ctx_len, group: int, kv_heads: int, window: int = 0,
                               target_waves: int = TARGET_WAVES, head_dim: int = 0,
                               min_split_keys: int = MIN_SPLIT_KEYS, block_tiles=TILES_PER_BLOCK // 2,
                               most_keys: int = WHOLE) -> AttentionWork:
    """``head_dim``: 0 keeps every item on the one-wavefront kernel (callers that do not know it).

    Items with at least half a block of tiles (prompt portions) go to the block kernel, the others
    keep one wavefront per tile.  In both classes the keys are cut into ranges when the class alone
    would not fill the chip; the number of ranges of an item follows its context, so that a long
    context beside short ones does not become the one long-running unit.  Where the single wavefronts fill the chip
    without ranges, ``most_keys`` is the most that one of them goes through."""
    q_len = np.asarray(q_len, dtype=np.int64)
    ctx_len = np.asarray(ctx_len, dtype=np.int64)
    if ((q_len < 1) | (q_len > ctx_len)).any():
        raise ValueError(_BAD_LENGTHS)
    q_start = np.concatenate(([0], np.cumsum(q_len)[:-1]))      # items' tokens lie one after the other
    tiles = (q_len * group + 15) // 16
    reach = np.minimum(ctx_len, window + q_len) if window else ctx_len      # keys an item's tiles can read
    in_blocks = items_in_blocks(q_len, group, head_dim, block_tiles)

    def keys_per_unit(units_per_item, wanted: int, least: int, most: int = WHOLE) -> int:
        """Keys of a range so that all ranges together number about ``wanted``."""
        in_flight = int(units_per_item.sum()) * kv_heads
        if in_flight >= wanted:
            return most
        if int((units_per_item * (reach // least)).sum()) * kv_heads < wanted // 2:
            least = max(32, least // 2)
        share = -(-int((units_per_item * reach).sum()) * kv_heads // wanted)
        return max(least, -(-share // 32) * 32)

    nblocks = np.where(in_blocks, -(-tiles // TILES_PER_BLOCK), 0)
    alone = np.where(in_blocks, 0, tiles)
    # blocks of an item whose portion is most of what it reads (a whole prompt) are never cut: they take
    # their places among the blocks wanted as they are
    cut = in_blocks & (reach - q_len >= PREFIX_PER_PORTION * q_len)
    whole = int(np.where(cut, 0, nblocks).sum()) * kv_heads
    block_keys = keys_per_unit(np.where(cut, nblocks, 0), TARGET_BLOCKS - whole, MIN_BLOCK_KEYS) if TARGET_BLOCKS > whole else 1 << 30
    keys = np.where(in_blocks, np.where(cut, block_keys, 1 << 30), keys_per_unit(alone, target_waves, min_split_keys, most_keys))
    # equal ranges (multiples of 32 keys) over [first_key, ctx) of every item
    first_key = np.maximum(0, ctx_len - reach) // 32 * 32
    span = ctx_len - first_key
    splits = np.clip(-(-reach // keys), 1, MAX_SPLITS)
    chunk = -(-(-(-span // splits)) // 32) * 32
    splits = np.where(splits > 1, -(-span // np.maximum(chunk, 1)), 1)
    chunk = np.where(splits > 1, chunk, span)
    # partial slots: tile t, range s of an item -> base + t * splits + s, for items with several ranges
    slots_of = np.where(splits > 1, tiles * splits, 0)
    base = np.cumsum(slots_of) - slots_of
    num_slots = int(slots_of.sum())

    def expand(rows_per_item, fields: int, tiles_per_row: int):
        """One record per (row, range) of every item: rows are tiles or runs of tiles."""
        if not rows_per_item.any():
            return np.zeros((0, fields), dtype=np.int32), None
        count = rows_per_item * splits
        item = np.repeat(np.arange(len(tiles)), count)
        j = np.arange(int(count.sum())) - np.repeat(np.cumsum(count) - count, count)
        row, s = j // splits[item], j % splits[item]
        out = np.zeros((item.size, fields), dtype=np.int32)
        out[:, 0], out[:, 1] = item, row * tiles_per_row
        begin = first_key[item] + s * chunk[item]
        out[:, 2], out[:, 3] = begin, np.minimum(begin + chunk[item], ctx_len[item])
        out[:, 4] = np.where(splits[item] > 1, base[item] + row * tiles_per_row * splits[item] + s, -1)
        out[:, 5], out[:, 6], out[:, 7] = q_start[item], q_len[item], ctx_len[item]
        return out, item

    units, _ = expand(alone, UNIT_FIELDS, 1)
    blocks, block_item = expand(nblocks, BLOCK_UNIT_FIELDS, TILES_PER_BLOCK)
    if block_item is not None:
        blocks[:, 8] = splits[block_item]
    tasks = np.zeros((0, TASK_FIELDS), dtype=np.int32)
    if num_slots:
        merged = np.nonzero(splits > 1)[0]
        count = tiles[merged]
        item = np.repeat(merged, count)
        tile = np.arange(int(count.sum())) - np.repeat(np.cumsum(count) - count, count)
        tasks = np.zeros((item.size, TASK_FIELDS), dtype=np.int32)
        tasks[:, 0], tasks[:, 1], tasks[:, 2] = item, tile, base[item] + tile * splits[item]
        tasks[:, 3], tasks[:, 4], tasks[:, 5] = splits[item], q_start[item], q_len[item]

    if len(blocks):
        # longest first: a block's work grows with the position of its rows, and the blocks that are
        # started last decide when the kernel ends
        pos0 = ctx_len - q_len
        last_key = pos0[blocks[:, 0]] + ((blocks[:, 1].astype(np.int64) + TILES_PER_BLOCK) * 16 - 1) // group
        end = np.minimum(np.minimum(last_key + 1, ctx_len[blocks[:, 0]]), blocks[:, 3])
        begin = blocks[:, 2].astype(np.int64)
        if window:
            begin = np.maximum(begin, pos0[blocks[:, 0]] + (blocks[:, 1].astype(np.int64) * 16) // group - window + 1)
        blocks = blocks[np.argsort(-np.maximum(end - begin, 0), kind="stable")]
    return AttentionWork(units, tasks, num_slots, blocks)
