"""Which requests of a batch hold the same committed rows, and the plan that attends those
rows once for all of them.

Lineage.  The rows of a request are its own from some position on; the rows below were
copied from another request (PersistentTargetKV.share_prefix).  A lineage lists, in order,
(origin, end): rows up to `end` were written by `origin`, the last span (its own rows) having
no end.  Committed rows never change, so two requests hold the same rows up to the
position where their lineages part.

Groups.  A request is in one group at most, whose members share the rows that all of them
hold: of a system prompt for many and a document for some of these, each request
shares one or the other, by what saves more rows (shared_groups).

Plan.  Runs and prompt columns over each request's own keys, as in a mixed plan
(schedule.mixed_plan), whose records start at the prefix's end, with partial slots for the
prefix's segments ahead of the request's own; and a list of prefix items
(dspark_shared_attn_fwd in include/dspark_amd.h).  A request of a group always
has partials, at least one of the prefix and one of its own keys.
"""
from collections import namedtuple

import numpy as np

from .schedule import (DECODE_TOKENS, MIN_SEGMENT, PART_TILE_BYTES, PROMPT_TOKENS, REQ_INTS, RESIDENT_PER_CU, SEGMENT_COST,
                       TILE, WORK_INTS, XCDS, _balanced_runs, _prompt_columns, prompt_segments, run_count, run_shares)

PREFIX_TILE = 64              # prefixes end, and are cut, at multiples of this many keys (a ring stage)
# Fewest key rows that a group must save to be one: sharing takes partials and a second part.
# Shared / each request its own copy, us a call: 2 requests of 7 tokens over 1,000 rows
# 12.2 / 11.4, 4 over 1,000 12.2 / 11.9, 2 over 4,100 15.0 / 17.2, 16 over 2,000 17.5 / 28.6, 64 over 64
# 14.5 / 12.6, over 128 15.0 / 15.2, over 8,192 56 / 353.
MIN_SAVED = 4096
# Groups of more than 32 tokens a request on average are bound by their products, not by
# reading rows: there the prefix's length decides, whose tiles pay for the partials of so many
# tokens.  Alike: 2 prompts of 40 over 800 rows 13.5 / 17.4, 2 of 400 over 800 25.2 / 31.0, 8 of 100 over
# 800 20.5 / 28.2, 16 of 200 over 768 59.7 / 58.6, over 512 53 / 47, over 256 48 / 36, 64 of 40 over
# 256 42 / 39, 4 of 400 over 800 38.2 / 34.6, over 1,200 44.1 / 43.4, 12 of 220 over 6,000 165 / 234.
MANY_TOKENS, MIN_LONG_ROWS = 32, 768
# Prefix workgroups per CU, in the kernel's grid.  Their segments are counted for one: beside
# them on a CU is a run of the requests' own keys, which memory bounds.  Segments for one / two
# per CU, us a call: 64 requests of 1 to 8 tokens over 8,192 rows and up to 1,024 own 57 / 61, 8
# of 7 over 16,384 27 / 38, 64 of 8 over 16,384 112 / 107, 12 prompts over 6,000 162 / 166.
PREFIX_PER_CU = 2
MIN_PREFIX_SEGMENT = 128      # fewest keys of a prefix segment
MAX_PREFIX_SEGMENTS = 32
# A segment's fixed work (its start, partials and their merge), in keys.  With 192 and 400: 6
# prompts of up to 100 tokens over 2,000 rows 27 and 22 us, 3 of 400 over 3,000 65 and 61, 64 requests
# over 8,192 56 and 57.
PREFIX_SEGMENT_COST = 400
# What each further segment costs a group, in keys, and with each of its token tiles: its
# partials, written and merged.  Without / with it, segments and us a call: 16 requests x 7 tokens
# over 2,000 rows 8 20.1 / 6 18.4, 12 of 2 groups over 3,056 14 and 17 19.8 / 8 16.3, 4 of 1 token over
# 10,403 32 39.0 / 15 36.2, 3 prompts of up to 400 over 3,000 3 56.5 / 2 52.7, 64 requests over 8,192
# the same 3.
PREFIX_PART_COST = 40, 6
# More room than PREFIX_TILES does not help prompts: 12 of 2 groups over 6,000 rows in 1, 2
# and 3 segments 165, 171 and 176 us.
PREFIX_TILES = 512            # partial tiles that prefix segments may take (more where one segment each needs it)
TOKEN_INTS = 4
MAX_BRANCHES = 16             # forks below forks that are looked at for groups of their own

SharedCapacity = namedtuple('SharedCapacity', 'run_records prompt_records runs requests columns tiles prefix_tiles items '
                                              'tokens')
Group = namedtuple('Group', 'members length slot')


# -- lineages ---------------------------------------------------------------------
def common_rows(a, b):
    """Rows that two lineages have in common from the start (None: no end)."""
    rows = 0
    for (origin, end), (other, other_end) in zip(a, b):
        if origin != other:
            break
        if end is None and other_end is None:
            return None
        rows = min(x for x in (end, other_end) if x is not None)
        if end != other_end:
            break
    return rows


def inherited(lineage, rows, origin):
    """The lineage of `origin` with its first `rows` rows copied from `lineage`'s."""
    spans = []
    for at, end in lineage:
        if rows <= (spans[-1][1] if spans else 0):
            break
        spans.append((at, rows if end is None else min(end, rows)))
    return (*spans, (origin, None))


def shared_groups(lineages, contexts, slots, query_lengths=None):
    """[Group(members, rows, slot)] of a batch: the requests of each group hold
    the same first `rows` rows, a multiple of PREFIX_TILE, which are read from `slot`.
    query_lengths: the requests' tokens (default: few)."""
    queries = query_lengths or [1] * len(lineages)
    families = {}
    for r, lineage in enumerate(lineages):
        families.setdefault(lineage[0][0], []).append(r)
    groups = []
    for members in families.values():
        if len(members) > 1:
            groups += _groups_from(lineages, contexts, queries, members, 0, 0)
    return [Group(sorted(members), rows, slots[min(members)]) for members, rows in groups]


def _saved(groups):
    return sum((len(members) - 1) * rows for members, rows in groups)


def _groups_from(lineages, contexts, queries, members, depth, branches):
    """Groups among requests whose lineages are the same up to span `depth`, whose origin they
    have in common too: all of them there, or those of a branch whose lineages stay the
    same for longer apart from the rest, whichever saves more rows."""
    while True:
        deeper = {}
        for r in members:
            if depth + 1 < len(lineages[r]):
                deeper.setdefault((lineages[r][depth][1], lineages[r][depth + 1][0]), []).append(r)
        if len(deeper) != 1 or len(*deeper.values()) < len(members):
            break
        depth += 1                                             # nobody leaves here
    reach = {r: contexts[r] if lineages[r][depth][1] is None else min(contexts[r], lineages[r][depth][1]) for r in members}
    chosen, here = [], _groups_at(members, reach, queries)
    for branch in deeper.values():
        if len(branch) < 2 or branches == MAX_BRANCHES:
            continue
        apart = _groups_from(lineages, contexts, queries, branch, depth + 1, branches + 1)
        inside = {r for group, _ in apart for r in group}
        rest = [r for r in members if r not in inside]
        without = _groups_at(rest, reach, queries)
        if apart and _saved(apart) + _saved(without) > _saved(here):
            members, here = rest, without
            chosen += apart
    return chosen + here


def _pays(members, rows, queries):
    if sum(queries[r] for r in members) > MANY_TOKENS * len(members):
        return rows >= MIN_LONG_ROWS
    return (len(members) - 1) * rows >= MIN_SAVED


def _groups_at(members, reach, queries):
    """[(members, rows)] of requests that have all rows in common up to where each one's reach
    ends: those who would shorten a group more than they gain stay out of it."""
    groups, members = [], sorted(members, key=lambda r: (-reach[r], r))
    while len(members) > 1:
        best = max(range(2, len(members) + 1), key=lambda n: (n - 1) * (reach[members[n - 1]] // PREFIX_TILE))
        rows = reach[members[best - 1]] // PREFIX_TILE * PREFIX_TILE
        if rows == 0 or not _pays(members[:best], rows, queries):
            break
        groups.append((members[:best], rows))
        members = members[best:]
    return groups


# -- plans ------------------------------------------------------------------------
def _width(query_length):
    """Partial tiles of a segment of a request."""
    return -(-int(query_length) // DECODE_TOKENS)


def shared_capacity(n_req, query_tokens, max_q, n_cu):
    """The regions of a fixed-capacity shared list (SharedCapacity)."""
    slots = max(XCDS, RESIDENT_PER_CU * n_cu // 8 // XCDS * XCDS)
    prompts = max_q > DECODE_TOKENS
    width = n_req + (query_tokens // DECODE_TOKENS if prompts else 0)
    prefix = max(width, min(PREFIX_TILES, MAX_PREFIX_SEGMENTS * width))
    own = width + n_req + slots + (PROMPT_TOKENS // DECODE_TOKENS * slots if prompts else 0)
    tiles = query_tokens // PROMPT_TOKENS + n_req                      # 32-token tiles at most
    return SharedCapacity(n_req + slots - 1, n_req + slots - 1 if prompts else 0, slots, n_req,
                          max(slots, RESIDENT_PER_CU * n_cu // 8, tiles) if prompts else 0, own + prefix, prefix, prefix + tiles, query_tokens)


def mixed_part_ints(c):
    """int32 of the mixed list's part, whole 32-byte records."""
    n = WORK_INTS * (c.run_records + c.prompt_records) + c.runs + 1 + REQ_INTS * c.requests + 2 * c.columns
    return -(-n // WORK_INTS) * WORK_INTS


def shared_ints(c):
    """int32 length of a shared list: the mixed list, then the prefix items."""
    return mixed_part_ints(c) + WORK_INTS * (1 + c.items) + TOKEN_INTS * c.tokens


def shared_bytes(c):
    return PART_TILE_BYTES * c.tiles


def prefix_columns(per_cu):
    """Prefix workgroups per KV head, for `per_cu` CUs per KV head."""
    return PREFIX_PER_CU * per_cu


def prefix_segments(tiles, rows, columns, room):
    """Segments of a group's prefix, for `tiles` token tiles per segment on `columns` workgroup
    slots per KV head: of those that keep MIN_PREFIX_SEGMENT keys each and fit `room`
    partials, the number whose rounds of slots and partials take the least time."""
    most = max(1, min(rows // MIN_PREFIX_SEGMENT, MAX_PREFIX_SEGMENTS, room))
    part = PREFIX_PART_COST[0] + PREFIX_PART_COST[1] * tiles
    return min(range(1, most + 1), key=lambda p: -(-tiles * p // columns) * (rows / p + PREFIX_SEGMENT_COST) + p * part)


def shared_plan(query_lengths, key_lengths, starts, groups, n_cu, capacity, *, xcd_speed=None, slot_balance=True):
    """The list of a batch whose `groups` share prefixes, laid out in the regions of
    `capacity` (an int32 array)."""
    c = capacity
    n = len(query_lengths)
    own_from = [0] * n
    for group in groups:
        for r in group.members:
            own_from[r] = group.length
    own = [k - f for k, f in zip(key_lengths, own_from)]
    q0 = np.concatenate(([0], np.cumsum(query_lengths))).tolist()
    width = [_width(q) for q in query_lengths]

    # the prefixes' segments: the groups share the columns by their work, and the room for partials
    per_head = max(1, n_cu // 8)
    work = [sum(query_lengths[r] for r in group.members) * group.length for group in groups]
    least = sum(width[r] for group in groups for r in group.members)
    parts, prefix_parts, items, tokens = [], [0] * n, [], []
    for group, cost in zip(groups, work):
        wide = sum(width[r] for r in group.members)
        share = max(1, per_head * cost // sum(work))
        room = max(1, c.prefix_tiles * wide // least // wide)
        p = prefix_segments(-(-sum(query_lengths[r] for r in group.members) // PROMPT_TOKENS), group.length, share, room)
        parts.append(p)
        for r in group.members:
            prefix_parts[r] = p

    # the requests' own keys
    decode = [r for r in range(n) if query_lengths[r] <= DECODE_TOKENS]
    prompts = [r for r in range(n) if query_lengths[r] > DECODE_TOKENS]
    # behind a prefix a request may have a few keys: each is worth a run of its own all the
    # same (by the keys alone 64 requests of 1 token would share 8 runs: 30 us a call)
    groups_of_runs = min(run_count(sum(max(own[r], MIN_SEGMENT) for r in decode) // (2 if prompts else 1), n_cu),
                         max(XCDS, n_cu // 8 // XCDS * XCDS) if prompts else c.runs)
    per_run = [[] for _ in range(XCDS)]
    if decode:
        per_run = [[(decode[r], a, b) for r, a, b in run]
                   for run in _balanced_runs([own[r] for r in decode], groups_of_runs, TILE, SEGMENT_COST,
                                             shares=run_shares(groups_of_runs, xcd_speed, n_cu if slot_balance else None))]
    held = [0] * n
    for run in per_run:
        for r, _, _ in run:
            held[r] += 1
    taken = sum(p * width[r] for r, p in enumerate(prefix_parts)) + sum(held) + sum(width[r] for r in prompts)
    loose = [(prompts[i], a, b) for i, a, b in
             prompt_segments([query_lengths[r] for r in prompts], [own[r] for r in prompts],
                             max(0, c.prompt_records - len(prompts)), n_cu, c.tiles - taken)]
    segs = [x for run in per_run for x in run] + loose
    for r, _, _ in loose:
        held[r] += 1
    slot, used = [-1] * n, 0
    for r in range(n):
        if prefix_parts[r] + held[r] > 1:
            slot[r] = used
            used += (prefix_parts[r] + held[r]) * width[r]
    nxt = [s + p * w for s, p, w in zip(slot, prefix_parts, width)]
    records = []
    for r, a, b in segs:
        at = -1
        if slot[r] >= 0:
            at, nxt[r] = nxt[r], nxt[r] + width[r]
        records += (r, own_from[r] + a, own_from[r] + b, at, q0[r], query_lengths[r], key_lengths[r], starts[r])
    requests = []
    for r in range(n):
        requests += (max(slot[r], 0), prefix_parts[r] + held[r], q0[r], query_lengths[r])
    ranges = [0]
    for run in per_run:
        ranges.append(ranges[-1] + len(run))
    first = ranges[-1]
    rows = [(r, q0[r], query_lengths[r], key_lengths[r], starts[r]) for r in prompts]
    place = {r: i for i, r in enumerate(prompts)}
    columns = _prompt_columns(rows, [(place[r], own_from[r] + a, own_from[r] + b) for r, a, b in loose], c.run_records, True)

    start = 0
    for group, p in zip(groups, parts):
        m = np.array(group.members)
        q, w, s = (np.array([x[r] for r in group.members], dtype=np.int32) for x in (query_lengths, width, slot))
        count = int(q.sum())
        ends = np.cumsum(q, dtype=np.int32)
        t = np.arange(count, dtype=np.int32) - np.repeat(ends - q, q)          # the token's place in its request
        rows = np.array(q0, dtype=np.int32)[m]
        tokens.append(np.stack((np.repeat(rows, q) + t, np.repeat(s, q) + t // DECODE_TOKENS, t % DECODE_TOKENS,
                                np.repeat(w, q)), 1))
        tile = np.arange(0, count, PROMPT_TOKENS, dtype=np.int32)
        cuts = np.arange(p + 1, dtype=np.int32) * (group.length // PREFIX_TILE) // p * PREFIX_TILE
        some = np.zeros((p, len(tile), WORK_INTS), dtype=np.int32)           # all token tiles of a segment together
        some[:, :, 0], some[:, :, 3] = group.slot, np.arange(p)[:, None]
        some[:, :, 1], some[:, :, 2] = cuts[:-1, None], cuts[1:, None]
        some[:, :, 4], some[:, :, 5] = start + tile, np.minimum(PROMPT_TOKENS, count - tile)
        items.append(some.reshape(-1, WORK_INTS))
        start += count
    items = np.concatenate(items).reshape(-1) if items else ()
    tokens = np.concatenate(tokens).reshape(-1) if tokens else ()

    if (first > c.run_records or len(loose) > c.prompt_records or len(per_run) > c.runs or n > c.requests
            or len(columns) > 2 * c.columns or used > c.tiles or len(items) > WORK_INTS * c.items
            or len(tokens) > TOKEN_INTS * c.tokens):
        raise ValueError('Segment plan exceeds its fixed capacity')
    out = np.zeros(shared_ints(c), dtype=np.int32)
    cut, n_work = WORK_INTS * first, c.run_records + c.prompt_records
    after, base = WORK_INTS * n_work + c.runs + 1, mixed_part_ints(c)
    for at, part in ((0, records[:cut]), (WORK_INTS * c.run_records, records[cut:]),
                     (WORK_INTS * n_work, ranges + [first] * (c.runs - len(per_run))), (after, requests),
                     (after + REQ_INTS * c.requests, columns), (base, [len(items) // WORK_INTS]), (base + WORK_INTS, items),
                     (base + WORK_INTS * (1 + c.items), tokens)):
        out[at:at + len(part)] = part
    return out
