"""Items of PreparedBlockAttention's split launches, by the plan that its entry
and its kernel make: their states never pass the scratch.  Without a device."""
import random

import pytest

from tests.test_block_cache_host import good_attention, scratch

SLOTS, KEYS, MAX_SPLIT_WORK = 512, 64, 0x1ffffff
MIN_TILES = {1: 1, 2: 2, 4: 8}


def scratch_of(tokens, heads, kv_heads, batch, width, cmp_width, ratio, window):
    """(rows of a unit / 16, units, work-groups) of a split launch as its scratch has room for; None where it is not split."""
    a = good_attention()
    a.tokens, a.heads, a.kvHeads, a.batch, a.ratio, a.window = tokens, heads, kv_heads, batch, ratio, min(window, 2 ** 32 - 1)
    a.oriTableWidth, a.cmpTableWidth = width, cmp_width
    a.oriStride = a.cmpStride = 16384 * kv_heads
    ok, partial, units = scratch(a)
    assert ok == 0
    if not partial:
        return None
    rows, group, near = tokens * heads, heads // kv_heads, window + 128
    tiles = ((cmp_width + 1) // 2 if ratio > 1 else 0) + (min(near // 32, width) + 1) // 2
    each, score = -(-(rows // kv_heads) // batch), ((rows + 63) // 64) ** 2 * tiles
    wide = score >= 400000 or score >= 130000 and tiles >= 128
    rt = 1 if each <= 16 or score < 8000 else 2 if each <= 32 or not wide else 4
    most = min(rows // (16 * rt) + batch * kv_heads, tokens * kv_heads * -(-group // (16 * rt))) + 1
    grid = -(-min(SLOTS, most * tiles) // 8) * 8
    assert (partial, units) == (grid * 16 * rt * 514 * 4, 32 * (1 + most))
    return rt, most, grid


def items_of(rt, units, new, lengths, heads, kv_heads, width, cmp_width, ratio, window, pad, by_all=True):
    """Items of the plan, None where it splits nothing; `by_all` False: the last try by the units' average tiles."""
    rows, group, requests, work, most = 16 * rt, heads // kv_heads, [], 0, 0
    seen = lambda p: min(max(p + 1, 0) // ratio, cmp_width * 32) if ratio > 1 else 0  # noqa: E731
    for count, length in zip(new, lengths):
        per_head = -(-count * group // rows)
        tiles = 0
        if length > 0 and count > 0:
            reach = min(length, width * 32, window + (rows - 1) // group + 1 + 32)
            compressed = seen(length - 1)
            tiles = -(-compressed // KEYS) - (-reach // KEYS)
            less = min(reach, max(0, count - (length - reach))) + compressed - seen(length - count)
            work += min(per_head * kv_heads * max(1, tiles - less // (2 * KEYS)), MAX_SPLIT_WORK)
            most += min(per_head * kv_heads * tiles, MAX_SPLIT_WORK)
        requests.append((per_head * kv_heads, tiles))
    padding = -(-pad * heads // rows)
    whole = sum(u for u, _ in requests) + padding
    if whole > units:
        return None
    items = lambda each: sum(u * max(1, -(-t // each)) for u, t in requests) + padding  # noqa: E731
    share = lambda tiles, room: max(MIN_TILES[rt], -(-tiles // room))  # noqa: E731
    tries = [share(work, SLOTS - whole * i // 3) for i in range(4)]
    if len(new) <= 64:
        for each in tries if by_all else tries[:3]:
            if items(each) <= SLOTS:
                return items(each)
    return items(share(most, SLOTS - whole) if by_all else tries[3])


# Prompts into empty caches: a request's first units see far fewer tiles than its last.
PROMPTS = [
    dict(new=[522], lengths=[528], heads=8, kv_heads=4, ratio=1, window=1000),
    dict(new=[739], lengths=[739], heads=6, kv_heads=2, ratio=1, window=2 ** 30),
    dict(new=[262], lengths=[268], heads=6, kv_heads=2, ratio=128, window=2 ** 30),
    dict(new=[278], lengths=[278], heads=20, kv_heads=4, ratio=1, window=2 ** 30),
    dict(new=[30, 771, 1, 120], lengths=[30, 771, 1, 120], heads=3, kv_heads=1, ratio=1, window=2 ** 30),
    dict(new=[771] + [1] * 69, lengths=[771] + [9] * 69, heads=3, kv_heads=1, ratio=1, window=2 ** 30),
]


def planned(c, by_all):
    width, cmp_width = max(c["lengths"]) // 32 + 1, max(c["lengths"]) // (32 * c["ratio"]) + 1
    args = (c["heads"], c["kv_heads"])
    fits = scratch_of(sum(c["new"]), *args, len(c["new"]), width, cmp_width, c["ratio"], c["window"])
    assert fits
    rt, units, room = fits
    return items_of(rt, units, c["new"], c["lengths"], *args, width, cmp_width, c["ratio"], c["window"], 0, by_all), room


@pytest.mark.parametrize("case", PROMPTS, ids=lambda c: f"{c['new'][0]}x{len(c['new'])}_{c['heads']}_{c['kv_heads']}")
def test_prompts_stay_in_the_scratch(case):
    items, room = planned(case, True)
    assert items is not None and items <= room


def test_average_tiles_would_not_do():
    """These prompts tell a plan by the units' average tiles from one by all of them."""
    assert all(items > room for items, room in (planned(c, False) for c in PROMPTS))


def test_items_never_pass_the_scratch():
    rng = random.Random(3)
    split = 0
    for _ in range(20000):
        kv_heads = rng.choice([1, 1, 2, 4])
        heads = kv_heads * rng.choice([1, 2, 3, 5, 8, 16, 32])
        most = rng.choice([1, 4, 40, 200, 800])
        new = [rng.randint(0, most) for _ in range(rng.choice([1, 1, 2, 4, 16, 65, 200]))]
        lengths = [0 if rng.random() < 0.05 else t + int(rng.choice([0, 0, 10, 300, 4000]) * rng.random()) for t in new]
        ratio, pad = rng.choice([1, 1, 128, 2]), rng.choice([0, 0, 3])
        window = rng.choice([1, 128, 1000, 2 ** 30])
        width = max(1, max(lengths) // 32 + rng.choice([0, 1, 5]))
        cmp_width = max(1, max(lengths) // (32 * ratio) + 1)
        if not sum(new) + pad:
            continue
        fits = scratch_of(sum(new) + pad, heads, kv_heads, len(new), width, cmp_width, ratio, window)
        if fits:
            rt, units, room = fits
            items = items_of(rt, units, new, lengths, heads, kv_heads, width, cmp_width, ratio, window, pad)
            assert items is None or items <= room
            split += items is not None
    assert split > 5000
