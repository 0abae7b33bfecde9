"""OSCAR configuration: environment names, derived byte sizes, split/grid policy.

Mirrors ``oscar_ascend/config.py`` (reference) value for value: the same environment
variable names, validation rules and derived sizes, so a deployment can switch packages
without touching its environment. One clip mode is added (``search``, the BASELINE
8-factor MSE search) and split policies for MI355X (``choose_splits_mi355x``,
``choose_history_partition`` for the token-bounded split rule with a host-side length, and
``choose_device_partition`` for the device rule, whose split length the GPU derives from
the step's lengths); the reference's ``choose_splits`` keeps its exact values.
"""

from __future__ import annotations

import functools
import math
import os
from dataclasses import dataclass

# Clip modes as passed across the C ABI.
CLIP_MODES = {"percentile": 0, "factor": 1, "search": 2}


@dataclass(frozen=True)
class OscarConfig:
    """Reference: oscar_ascend/config.py:8-81 (defaults 10-23, validation 25-43)."""

    head_dim: int = 256
    group_size: int = 256
    sink_tokens: int = 64
    recent_tokens: int = 256
    speculative_tokens: int = 3
    k_clip_ratio: float = 0.96
    v_clip_ratio: float = 0.92
    clip_mode: str = "percentile"
    k_clip_factor: float = 1.0
    v_clip_factor: float = 1.0
    k_rotation_path: str = ""
    v_rotation_path: str = ""
    block_n: int = 32
    queries_per_tile: int = 4

    def __post_init__(self):
        for ok, message in _config_rules(self):
            if not ok:
                raise ValueError(message)

    @property
    def data_bytes(self):
        """Packed code bytes per vector: four 2-bit codes per byte."""
        return self.head_dim // 4

    @property
    def vector_bytes(self):
        """Codes plus fp16 scale and fp16 zero."""
        return self.data_bytes + 4

    @property
    def slot_bytes(self):
        """K and V vectors of one token-head, rounded up to a 32-byte multiple (160)."""
        return ((2 * self.vector_bytes + 31) // 32) * 32

    @property
    def ring_tokens(self):
        return self.recent_tokens + self.speculative_tokens + 1

    @property
    def window_tokens(self):
        return self.sink_tokens + self.ring_tokens

    @classmethod
    def from_env(cls, speculative_tokens=3):
        """Reference: config.py:65-81 (same variable names and defaults)."""
        return cls(
            group_size=int(os.getenv("VLLM_OSCAR_GROUP_SIZE", "256")),
            sink_tokens=int(os.getenv("VLLM_OSCAR_SINK_TOKENS", "64")),
            recent_tokens=int(os.getenv("VLLM_OSCAR_RECENT_TOKENS", "256")),
            speculative_tokens=speculative_tokens,
            k_clip_ratio=float(os.getenv("VLLM_OSCAR_K_CLIP_RATIO", "0.96")),
            v_clip_ratio=float(os.getenv("VLLM_OSCAR_V_CLIP_RATIO", "0.92")),
            clip_mode=os.getenv("OSCAR_ASCEND_CLIP_MODE", "percentile"),
            k_clip_factor=float(os.getenv("OSCAR_ASCEND_K_CLIP_FACTOR", "1")),
            v_clip_factor=float(os.getenv("OSCAR_ASCEND_V_CLIP_FACTOR", "1")),
            k_rotation_path=os.getenv("VLLM_OSCAR_K_ROTATION_PATH", ""),
            v_rotation_path=os.getenv("VLLM_OSCAR_V_ROTATION_PATH", ""),
            block_n=int(os.getenv("OSCAR_ASCEND_BLOCK_N", "32")),
            queries_per_tile=int(os.getenv("OSCAR_ASCEND_QUERY_TILE", "4")),
        )


def _config_rules(cfg):
    """Accept/reject rules of the reference (config.py:25-43), one (condition, error) each."""
    finite_ratios = all(math.isfinite(r) for r in (cfg.k_clip_ratio, cfg.v_clip_ratio))
    finite_factors = all(math.isfinite(f) for f in (cfg.k_clip_factor, cfg.v_clip_factor))
    return (
        (cfg.head_dim == 256 and cfg.group_size >= cfg.head_dim,
         "head_dim must be 256 with a single quantization group per vector"),
        (min(cfg.sink_tokens, cfg.recent_tokens, cfg.speculative_tokens) >= 0,
         "sink, recent and speculative token counts must be >= 0"),
        (cfg.speculative_tokens <= 15, "speculative token count is limited to 15"),
        (cfg.clip_mode in CLIP_MODES,
         "OSCAR_ASCEND_CLIP_MODE must be one of " + ", ".join(CLIP_MODES)),
        (finite_ratios and all(r == 0 or 0.875 <= r <= 1
                               for r in (cfg.k_clip_ratio, cfg.v_clip_ratio)),
         "clip percentiles must be 0 (off) or lie in [0.875, 1]"),
        (finite_factors and all(0 < f <= 1 for f in (cfg.k_clip_factor, cfg.v_clip_factor)),
         "clip factors must lie in (0, 1]"),
        (cfg.block_n in (16, 32), "OSCAR_ASCEND_BLOCK_N must be 16 or 32"),
        (cfg.queries_per_tile in (1, 2, 4), "OSCAR_ASCEND_QUERY_TILE must be 1, 2 or 4"),
    )


def choose_splits(num_requests, num_kv_heads, max_query_len):
    """Reference split policy (config.py:84-89): 1 split for long chunks, else 32/16/8."""
    if max_query_len > 16:
        return 1
    heads = num_requests * num_kv_heads
    for bound, splits in ((8, 32), (32, 16)):
        if heads <= bound:
            return splits
    return 8


def choose_splits_mi355x(num_tasks, num_kv_heads, max_query_len, max_seq_len=None,
                         compute_units=256, waves_per_cu=2, min_tokens_per_split=1024,
                         max_splits=256):
    """Split count for MI355X's 256 CUs.

    Enough (task, head, split) workgroups to give every CU ``waves_per_cu`` workgroups,
    but no split shorter than ``min_tokens_per_split`` history tokens when a host upper
    bound on the sequence length is known. Never reads device lengths. Long prefill
    chunks keep one split, as the reference does, to bound scratch.
    """
    if max_query_len > 16:
        return 1
    parallel = max(1, num_tasks * num_kv_heads)
    want = -(-compute_units * waves_per_cu // parallel)
    if max_seq_len is not None:
        want = min(want, max(1, max_seq_len // min_tokens_per_split))
    splits = 1
    while splits < want:
        splits *= 2
    return max(1, min(splits, max_splits))


def choose_history_partition(num_tasks, num_kv_heads, max_query_len, max_seq_len=None,
                             total_seq_len=None, slots=None, min_tokens_per_split=1024,
                             max_splits=256, rows=None, reserved=0):
    """``(splits, split_tokens)`` of the history branch on MI355X (no reference counterpart).

    Each request gets ceil(history / split_tokens) splits (token-bounded rule of
    ``kernels.attention_partials``), ``split_tokens`` sized so that the batch's history
    (``total_seq_len``, a host-side sum) fills ``slots`` workgroups, and ``splits`` is the
    longest request's share. ``slots`` defaults to 512 (two workgroups per CU) and, for tasks
    of more than 16 query rows (``rows``; the work-queue kernel, one workgroup per CU), to 448:
    about 1.8 units per CU, which measured best on the ragged MTP batch (units of 2816 tokens:
    106 us, 2432: 114-120 us, 3456: 116 us). A uniform batch gets the same partition as
    ``choose_splits_mi355x``; a ragged one stops waiting on its longest request. Without a
    host-side length bound it falls back to ``choose_splits_mi355x`` with the reference rule
    (split_tokens 0).

    ``reserved``: workgroup slots that other workgroups of the same launch hold (the
    pre-attention roles dispatched ahead of the history splits). The splits then fit in the
    remaining slots for any split of the lengths: a batch of ``num_tasks`` requests with
    ``total`` history tokens uses at most ``total / split_tokens + num_tasks`` splits per KV
    head. At c3 (48 role workgroups) this gives 14 splits of 2432 tokens: 50.7 us per layer
    step against 53.0 us with 16 splits, whose last workgroups waited for the roles' slots.
    """
    if slots is None:
        slots = 448 if rows is not None and rows > 16 else 512
    if max_query_len > 16 or max_seq_len is None:
        return choose_splits_mi355x(num_tasks, num_kv_heads, max_query_len, max_seq_len), 0
    if total_seq_len is None:
        total_seq_len = max_seq_len * num_tasks
    avail = max(1, slots - int(reserved))
    per_slot = -(-int(total_seq_len) * num_kv_heads // avail)
    if reserved:
        per_slot = max(per_slot, -(-int(total_seq_len) * num_kv_heads //
                                   max(1, avail - num_tasks * num_kv_heads)))
    split_tokens = max(min_tokens_per_split, -(-per_slot // 64) * 64)
    splits = min(max_splits, max(1, -(-int(max_seq_len) // split_tokens)))
    return splits, split_tokens


# Workgroup slots of the history launch on MI355X: two workgroups per CU for up to 16 query
# rows per task (256 CUs), and for the eight-wavefront work queue (17-32 rows) about 1.8 units
# per CU, which measured best on the ragged MTP batch.
HISTORY_SLOTS = 512
QUEUE_SLOTS = 448
# Bytes of split scratch one split slot costs per query row (fp32 partial row + LSE).
SPLIT_ROW_BYTES = 256 * 4 + 4


DEVICE_MIN_SPLIT = 1024


def device_split_tokens(history_total, tasks, num_kv_heads, budget, fit_grid=True):
    """The split length the history kernels derive on the GPU under the device rule
    (``split_tokens = -budget``), from the step's history tokens ``history_total`` over
    ``tasks`` tasks: max(1024, 64 * ceil(ceil(H * total / room) / 64)). ``fit_grid`` (the
    paired kernel's grid of unit slots, up to 8 query rows per task): room =
    max(1, budget - H * tasks), so that sum ceil(L / T) over the tasks stays within budget / H
    units per kv head; otherwise (a slot per split, or the work queue) room = budget."""
    room = max(1, int(budget) - (num_kv_heads * int(tasks) if fit_grid else 0))
    per = -(-num_kv_heads * int(history_total) // room)
    return int(min(max(-(-per // 64) * 64, DEVICE_MIN_SPLIT), 1 << 30))


def choose_device_partition(programs, num_kv_heads, max_query_len, tokens, q_heads,
                            queries_per_tile=4, reserved=0, max_splits=128,
                            scratch_bytes=128 << 20):
    """``(splits, split_tokens)`` of the device rule (no reference counterpart).

    Everything here is known when a graph is captured: the grid capacity ``programs``, the
    step's token count ``tokens`` and the launch form (``reserved`` workgroup slots held by
    the pre-attention roles of the same launch). The split length itself is derived on the GPU
    from the step's lengths (``split_tokens = -budget``, budget = the history launch's free
    workgroup slots), so one captured launch stays right and balanced at any context length,
    as the reference's host-count rule is (config.py:84-89), with token-bounded splits.

    ``splits`` bounds the splits of one request and sizes the split scratch. Up to 8 query
    rows per task it allows twice the even share of a batch of 32 requests or fewer
    (16 x ceil(32 / programs)), at least 16 (the one-round split merge), at most
    ``max_splits``; above 16 rows (the work queue, ragged MTP batches whose longest request
    takes a large share) it is bounded by ``scratch_bytes`` of split rows. A request that
    would need more splits gets longer ones. Steps with more than 16 query tokens in some request
    keep one split (config.py:86-87); above 8 rows per task their caller asks
    ``choose_chunk_splits`` instead.
    """
    if max_query_len > 16:
        return 1, 0
    rows = min(max(int(max_query_len), 1), queries_per_tile) * (q_heads // num_kv_heads)
    slots = QUEUE_SLOTS if rows > 16 else HISTORY_SLOTS
    budget = max(1, slots - int(reserved))
    if rows > 16:
        per_split = max(1, int(tokens) * q_heads * SPLIT_ROW_BYTES)
        splits = min(max_splits, max(16, scratch_bytes // per_split))
    else:
        splits = min(max_splits, 16 * max(1, -(-32 // max(1, int(programs)))))
    return splits, -budget


# Rows of a history tile of a continuation chunk, tokens of its pipeline step, and what a step, a
# workgroup's start and a merged split row cost on MI355X (us; one workgroup per CU).
CHUNK_TILE_ROWS, CHUNK_STEP_TOKENS = 128, 128
CHUNK_STEP_US, CHUNK_START_US, CHUNK_ROW_US = 4.0, 10.0, 5.5e-4


# The layers of a step ask with the same arguments: the two rules below are pure functions of a few
# integers, and the later layers' answers come from a bounded table (5 us of host time per layer in
# eager steps whose launches take 57).
@functools.lru_cache(maxsize=256)
def choose_chunk_splits(tokens, requests, num_kv_heads, q_heads, max_seq_len, compute_units=256,
                        max_splits=16, scratch_bytes=128 << 20):
    """Split count of a continuation chunk's history branch (more than 16 query tokens in some
    request; no reference counterpart, config.py:86-87 keeps one split).

    The launch has a workgroup per 128-row tile, KV head and split, one per CU at a time; a chunk
    of 2048 tokens x 6 heads is 96 tiles, which one split leaves on 96 of 256 CUs, and a decode
    request beside it is one tile of few rows. The count with the least modelled time of rounds
    over the CUs plus split rows written and merged, from host-side values (2048 tokens over
    32768: 980 / 522 / 432 / 423 / 473 us for 1 / 2 / 5 / 8 / 16 splits), at most 16 (the one-round
    split merge) and at most ``scratch_bytes`` of split rows, unless one split needs more: the
    engine's memory profile does not see the scratch of a step (8192 tokens x 12 heads over 131072
    would take 8 splits and 0.8 GB). One split when no host-side length is known."""
    if not max_seq_len:
        return 1
    group = q_heads // num_kv_heads
    tiles = num_kv_heads * (tokens * group // CHUNK_TILE_ROWS + max(1, requests))
    steps = -(-int(max_seq_len) // CHUNK_STEP_TOKENS)
    max_splits = max(1, min(max_splits, scratch_bytes // max(1, tokens * q_heads * SPLIT_ROW_BYTES)))

    def cost(splits):
        rounds = -(-tiles * splits // compute_units)
        return (rounds * (-(-steps // splits) * CHUNK_STEP_US + CHUNK_START_US)
                + tokens * q_heads * splits * CHUNK_ROW_US)

    return min(range(1, min(max_splits, steps) + 1), key=cost)


# The start of a workgroup among others of the launch, most of it beside their work.
CHUNK_SHORT_US = 6.0
# The task-shaped history kernels (us): a 64-token chunk of one task on its CU, and the share of a
# CU that it costs in a launch that fills them, with 16 query rows per task or fewer and with more.
TASK_CHUNK_US, TASK_LOAD_US = (0.45, 0.81), (0.45, 0.6)


@functools.lru_cache(maxsize=256)
def chunk_kernel_pays(tokens, requests, num_kv_heads, q_heads, splits, max_seq_len,
                      total_seq_len=None, total_query_keys=None, queries_per_tile=4,
                      compute_units=256):
    """Whether the 128-row-tile history kernel with ``splits`` splits takes less time than the
    task-shaped one with one split, in a step with more than 16 query tokens in some request (no
    reference counterpart). Host-side values: ``total_query_keys`` sums query tokens times length
    over the requests. False when no length is known.

    A request of one token is a whole tile of few rows (one CU at 3.7 us per 128 tokens, against
    1.6 for its task), so decodes beside a short chunk are better off as tasks, and so are short
    histories, whose split rows cost more than the history does. The tile kernel is taken where an
    upper estimate of its time (the load of all tiles and four fifths of its longest workgroup, or
    rounds of that) is below a lower one of the other's (its longest task, or the load of all
    tasks); unknown sums are taken at their worst for it. Layer step with the one and the other
    kernel (us): 2048 tokens over 32768, 5 splits 625 and 810, 1 split 1141 and 810; 64 over 16000
    beside 30 decodes of 2000 to 16000 tokens 150 and 258, beside 250 370 and 302; two KV heads,
    four query heads each, beside 60 313 and 183; 300 over 500 112 and 101. Over 226 steps the
    rule's kernel took at most 1.01 of the task-shaped one's time, 0.83 on average, and 1.02 of
    the faster one's."""
    if not max_seq_len:
        return False
    longest, group = int(max_seq_len), q_heads // num_kv_heads
    total = int(total_seq_len) if total_seq_len else requests * longest
    pairs = tokens * longest if requests == 1 else total_query_keys
    chunk_us, load_us = (us[queries_per_tile * group > 16] for us in (TASK_CHUNK_US, TASK_LOAD_US))
    # A request of q tokens has about (q + tile - 1) / tile tasks.
    task_tokens = (pairs + total * (queries_per_tile - 1)) / queries_per_tile if pairs else total
    task = max(chunk_us * longest / 64,
               load_us * num_kv_heads * task_tokens / 64 / compute_units)
    tiles = num_kv_heads * (tokens * group // CHUNK_TILE_ROWS + requests)
    tile_tokens = min(num_kv_heads * ((pairs or tokens * longest) * group / CHUNK_TILE_ROWS + total),
                      tiles * longest)
    longest_us = -(-longest // CHUNK_STEP_TOKENS // splits) * CHUNK_STEP_US + CHUNK_START_US
    rounds = tiles * splits / compute_units
    tile = min(tile_tokens / CHUNK_STEP_TOKENS / compute_units * CHUNK_STEP_US
               + rounds * CHUNK_SHORT_US + 0.8 * longest_us, math.ceil(rounds) * longest_us)
    if splits > 1:
        tile += tokens * q_heads * splits * CHUNK_ROW_US
    return tile < task


# Times of a layer step (us) by its query rows per history task, up to 8, 16 and 32, and of steps
# with more than 16 query tokens in a request: without a plan of shared prefixes (start, per million
# positions of a task's rows, per thousand query rows) and with it (start, per million positions of
# 16 rows that a request has to itself, the same of a group, per thousand query rows).
STEP_US = ((24.1, 23.3, 16.6), (42.3, 29.2, 8.9), (51.0, 40.2, 9.7), (73.3, 30.9, 3.6))
SHARED_STEP_US = ((33.6, 35.9, 23.5, 19.3), (39.4, 33.8, 20.2, 11.3), (47.0, 26.7, 17.9, 9.2),
                  (62.7, 18.9, 17.3, 5.8))


@functools.lru_cache(maxsize=256)
def shared_prefix_pays(tokens, requests, num_kv_heads, q_heads, max_query_len, total_seq_len=None,
                       saved_tokens=None, groups=1, total_query_keys=None, queries_per_tile=4):
    """Whether a layer step takes less time with the shared positions of its requests computed once
    (pre-attention, shared history, merge, post-attention) than with the history launch that carries
    the BF16 branch and the store (no reference counterpart). Host-side values: ``saved_tokens`` sums
    each group's shared tokens over its members but one; unknown, the groups share everything.
    ``total_query_keys`` sums query tokens times length. True when the lengths are not known: then
    the caller decides.

    A step with a plan is four launches and not three, and takes a request's own positions 16 rows at
    a time, so it pays where much is shared: 6 samples of 2000 tokens 24.3 us without and 33.1 with
    it, 32 of 32000 43.3 and 47.6, 256 of 32500 216 and 120; 64 requests of 16000 tokens with 4000 of
    them shared 51 and 67; 160 of 16000, 3 query tokens, 800 shared 183 and 238, 8000 shared 182 and
    160. Both times are estimated, linear in the positions and rows; the estimates are within a
    quarter of most measured times, so the plan is taken where its one is below 0.85 of the other.
    Over 890 steps of 1 to 4 KV heads and 4 to 8 query heads each the choice took at most 1.01 of the
    time without the plan, 0.96 on average (the faster one's each time: 0.91)."""
    if total_seq_len is None:
        return True
    requests, groups = max(1, requests), max(1, groups)
    if requests <= groups:
        return False
    group = q_heads // num_kv_heads
    if saved_tokens is None:
        saved_tokens = total_seq_len * (requests - groups) // requests
    once = saved_tokens * groups / (requests - groups)  # shared positions, each group's once
    own = max(0.0, total_seq_len - saved_tokens - once)
    queries = total_query_keys / max(1, total_seq_len) if total_query_keys else max_query_len
    rows = min(max_query_len, queries_per_tile) * group
    kind = 3 if max_query_len > 16 else 0 if rows <= 8 else 1 if rows <= 16 else 2
    tasks = math.ceil(queries / queries_per_tile)
    own_tiles = math.ceil(queries * group / 16)
    group_tiles = math.ceil(requests / groups * queries * group / 16)
    million, thousand = num_kv_heads / 1e6, tokens * q_heads / 1e3
    start, position, row = STEP_US[kind]
    without = start + position * total_seq_len * tasks * million + row * thousand
    start, alone, shared, row = SHARED_STEP_US[kind]
    return (start + (alone * own * own_tiles + shared * once * group_tiles) * million
            + row * thousand) < 0.85 * without


def choose_shared_slots(tokens, q_heads, most=256, scratch_bytes=128 << 20):
    """Partial rows per query row of a step with shared prefixes (no reference counterpart): the
    pieces that a row's positions may be cut into, four per lane of the wavefront that merges them
    and within ``scratch_bytes`` of rows, but at least 4."""
    return max(4, min(most, scratch_bytes // max(1, tokens * q_heads * SPLIT_ROW_BYTES)))


def percentile_selection(ratio, dim=256):
    """Descending ranks and interpolation weight of a linear quantile (config.py:92-97).

    Kept for API parity. The device kernels follow the torch.quantile arithmetic of the
    reference's test oracle (float32 rank, fused lerp), not this float64 weight.
    """
    position = ratio * (dim - 1)
    below, above = math.floor(position), math.ceil(position)
    return (dim - 1) - below, (dim - 1) - above, position - below


def task_capacity(tokens, requests, query_tile):
    """Upper bound on compact tasks (config.py:100-101)."""
    tiles_if_one_request = -(-tokens // query_tile)
    return min(tokens, tiles_if_one_request + requests - 1)


def attention_programs(tokens, requests, query_tile):
    """Grid size covering the compact task list (config.py:104-106)."""
    return max(1, task_capacity(tokens, requests, query_tile))
