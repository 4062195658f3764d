"""PreparedPathCommit, PreparedPageFork and PreparedPageCompact against plain
Python over lists; every table entry, count and byte equal."""
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
BLOCK, DIM = 32, 512


def say(*a):
    print(*a, file=sys.stderr, flush=True)


def ints(values):
    import torch
    return torch.tensor(np.asarray(values, np.int64).tolist(), dtype=torch.int32, device="cuda").reshape(np.shape(values))


def layered_pool(rng, pages, layers, rows=BLOCK, row=DIM, gap=0):
    """One backing of `layers` caches in each page (and a gap behind them), as numpy and as device views."""
    import torch
    stride = layers * rows * row + gap
    host = rng.integers(-128, 128, (pages, stride)).astype(np.int8)
    flat = torch.from_numpy(host.copy()).cuda()
    views = [flat.view(-1).as_strided((pages, rows, 1, row), (stride, row, row, 1), k * rows * row) for k in range(layers)]
    return host, flat, views


# ------------------------------------------------------------ paths

def plain_commit(host, layers, rows, row, table, cu, seq, paths, lens):
    out, pages = host.copy(), len(host)
    lengths = []
    cells = out[:, :layers * rows * row].reshape(pages, layers, rows, row)
    for b in range(len(seq)):
        nodes = cu[b + 1] - cu[b]
        if seq[b] <= 0:
            lengths.append(0)
            continue
        c, before, kept = max(0, seq[b] - nodes), -1, 0
        for k in range(max(0, min(lens[b], len(paths[b])))):
            node = paths[b][k]
            if not before < node < nodes:
                break
            before, kept = node, kept + 1
            place = []
            for at in (c + node, c + k):
                page = table[b][at // rows] if at // rows < len(table[b]) else -1
                place.append((page, at % rows) if 0 <= page < pages else None)
            if None not in place:
                cells[place[1][0], :, place[1][1]] = cells[place[0][0], :, place[0][1]]
        lengths.append(c + kept)
    return out, lengths


def random_paths(rng, nodes, depth):
    paths, lens = np.full((len(nodes), depth), -1, np.int64), []
    for b, n in enumerate(nodes):
        k = int(rng.integers(0, min(n, depth) + 1))
        paths[b, :k] = np.sort(rng.choice(n, k, replace=False))
        lens.append(k)
    return paths, lens


def commit_case(seed, nodes, committed, depth, layers=3, rows=BLOCK, row=DIM, gap=4096, width=None):
    rng = np.random.default_rng(seed)
    need = [-(-(c + n) // rows) for c, n in zip(committed, nodes)]
    pages = sum(need) + 2
    order = rng.permutation(pages)
    table, at = np.full((len(nodes), width or max(need)), -1, np.int64), 0
    for b, n in enumerate(need):
        held = min(n, table.shape[1])
        table[b, :held] = order[at:at + held]
        at += n
    paths, lens = random_paths(rng, nodes, depth)
    cu = np.concatenate([[0], np.cumsum(nodes)])
    seq = np.array(committed) + np.array(nodes)
    return rng, pages, table, cu, seq, paths, lens, layered_pool(rng, pages, layers, rows, row, gap)


def run_commit(host, flat, views, layers, rows, row, table, cu, seq, paths, lens):
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedPathCommit
    op = PreparedPathCommit(views, ints(table), ints(cu), ints(seq), ints(paths), ints(lens))
    assert op.run() is op.seq_lens
    torch.cuda.synchronize()
    want, lengths = plain_commit(host, layers, rows, row, table.tolist(), cu.tolist(), seq.tolist(), paths.tolist(), lens)
    np.testing.assert_array_equal(op.seq_lens.cpu().numpy(), lengths)
    np.testing.assert_array_equal(flat.cpu().numpy(), want)
    return op


@pytest.mark.parametrize("nodes,committed,depth", [
    ([1], [0], 1), ([8], [4096], 8), ([9, 1, 25, 64], [31, 32, 100, 5], 12), ([200], [63], 150),
    ([70, 3], [1, 0], 70)])
def test_commit(nodes, committed, depth):
    say(f"[commit] {nodes} {committed} depth {depth}")
    _, _, table, cu, seq, paths, lens, (host, flat, views) = commit_case(len(nodes), nodes, committed, depth)
    run_commit(host, flat, views, 3, BLOCK, DIM, table, cu, seq, paths, lens)


@pytest.mark.parametrize("rows,row,layers", [(32, 512, 38), (16, 48, 2), (1, 16, 1), (7, 1040, 5)])
def test_commit_other_pages(rows, row, layers):
    say(f"[commit] pages of {rows} x {row} bytes, {layers} caches")
    _, _, table, cu, seq, paths, lens, (host, flat, views) = commit_case(5, [9, 14], [40, 3], 9, layers, rows, row, 32)
    run_commit(host, flat, views, layers, rows, row, table, cu, seq, paths, lens)


def test_commit_keeps_what_it_reads():
    """Rows that are both written and read: every chain of moves over one another."""
    rng, _, table, cu, seq, paths, lens, (host, flat, views) = commit_case(6, [80, 80], [20, 21], 79)
    paths[0], lens[0] = np.arange(1, 80), 79                # each row moves down by one
    paths[1, :20], lens[1] = np.arange(3, 80, 4)[:20], 20
    say("[commit] overlapping moves")
    run_commit(host, flat, views, 3, BLOCK, DIM, table, cu, seq, paths, lens)


def test_commit_bad_paths_pages_and_padding():
    rng, pages, table, cu, seq, paths, lens, (host, flat, views) = commit_case(7, [9] * 9, [40] * 9, 9)
    paths[0, :4], lens[0] = [1, 3, 3, 5], 4                 # does not rise: two are kept
    paths[1, :3], lens[1] = [2, 9, 10], 3                   # no token of the request: one
    paths[2, :2], lens[2] = [-1, 2], 2                      # none
    paths[3, :2], lens[3] = [4, 6], 2 ** 31 - 1             # a length past the table: ends at -1
    paths[4, :2], lens[4] = [4, 6], -5
    seq[5] = 0                                              # graph padding
    table[6, 1] = pages                                     # rows on no page
    table[7, :] = -3
    seq[8] = 4                                              # fewer rows than tokens: nothing committed
    say("[commit] bad paths")
    run_commit(host, flat, views, 3, BLOCK, DIM, table, cu, seq, paths, lens)
    _, _, table, cu, seq, paths, lens, (host, flat, views) = commit_case(8, [9] * 2, [60] * 2, 9, width=2)
    say("[commit] a table too short")
    run_commit(host, flat, views, 3, BLOCK, DIM, table, cu, seq, paths, lens)


# ------------------------------------------------------------ fork

def plain_fork(host, used, table, seq, refs, parents, room, page_size):
    """(table, lengths, refs, missing, bytes) by the rules of the class."""
    rows, width, pages = len(table), len(table[0]), len(refs)
    out, new_refs = host.copy(), list(refs)
    for row in table:
        for page in row:
            if 0 <= page < pages:
                new_refs[page] -= 1
    free = [p for p in range(pages) if refs[p] == 0]
    seen, new, lengths, missing = set(), [], [], 0
    for parent in parents:
        entries = [-1] * width
        if not 0 <= parent < rows:
            new.append(entries)
            lengths.append(0)
            continue
        length = max(0, min(seq[parent], width * page_size))
        whole, needed = length // page_size, min(width, -(-(length + room) // page_size))
        first = parent not in seen
        seen.add(parent)
        for e in range(needed):
            old = table[parent][e]
            good = 0 <= old < pages
            if e < whole:
                entries[e] = old if good else -1
            elif first and good and refs[old] == 1:
                entries[e] = old
            elif not free:
                missing += 1
            else:
                entries[e] = free.pop(0)
                if e == whole and length % page_size and good:
                    out[entries[e], :used] = host[old, :used]
        if length % page_size and entries[whole] < 0:
            length = whole * page_size
        for page in entries:
            if page >= 0:
                new_refs[page] += 1
        new.append(entries)
        lengths.append(length)
    return new, lengths, new_refs, missing, out


def fork_state(rng, rows, width, longest, spare, layers=2, page_size=BLOCK, gap=4096, share=0.3):
    seq = rng.integers(0, longest + 1, rows)
    need = [-(-int(n) // page_size) for n in seq]
    total = sum(need)
    pages = total + spare
    order = rng.permutation(pages)
    table, at = np.full((rows, width), -1, np.int64), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    for b in range(1, rows):                                 # common prompts
        common = min(int(seq[b]) // page_size, int(seq[b - 1]) // page_size)
        if common and rng.random() < share:
            table[b, :common] = table[b - 1, :common]
    refs = np.bincount(table[table >= 0].ravel(), minlength=pages)
    free = np.flatnonzero(refs == 0)
    if len(free) > 2:
        refs[free[0]] = 3                                    # pages of another owner
    return table, seq, refs, layered_pool(rng, pages, layers, page_size, 64, gap)


def run_fork(state, parents, room, page_size=BLOCK, layers=2, flatten=False, inplace=False):
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedPageFork
    table, seq, refs, (host, flat, views) = state
    t, s, r = ints(table), ints(seq), ints(refs)
    caches, used = ([flat], flat.shape[1]) if flatten else (views, layers * page_size * 64)
    op = PreparedPageFork(caches, t, s, r, ints(parents), room=room, page_size=page_size,
                          output=(t, s, r) if inplace else None)
    new, lengths, counts = op.run()
    torch.cuda.synchronize()
    want = plain_fork(host, used, table.tolist(), seq.tolist(), refs.tolist(), list(parents), room, page_size)
    for got, expect in zip((new, lengths, counts, op.missing), want):
        np.testing.assert_array_equal(got.cpu().numpy().ravel(), np.asarray(expect).ravel())
    np.testing.assert_array_equal(flat.cpu().numpy(), want[4])
    if not inplace:
        np.testing.assert_array_equal(t.cpu().numpy(), table)
        np.testing.assert_array_equal(r.cpu().numpy(), refs)
    return op


@pytest.mark.parametrize("rows,children,width,longest,room", [
    (1, 1, 1, 32, 0), (1, 4, 60, 1900, 16), (1, 1, 5, 0, 0), (64, 64, 33, 1000, 16), (300, 277, 40, 900, 64),
    (5, 40, 600, 300, 9000), (37, 3, 12, 350, 1)])
def test_fork(rows, children, width, longest, room):
    rng = np.random.default_rng(rows + children)
    parents = rng.integers(-1, rows, children)
    say(f"[fork] {rows} rows to {children}, width {width}, room {room}")
    run_fork(fork_state(rng, rows, width, min(longest, width * BLOCK), 8 + children * (2 + room // BLOCK)), parents, room)


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("flatten", [False, True])
def test_fork_in_place_and_flat_backing(inplace, flatten):
    rng = np.random.default_rng(3)
    say(f"[fork] in place {inplace}, flat {flatten}")
    run_fork(fork_state(rng, 50, 30, 900, 200), rng.integers(-3, 53, 50), 40, flatten=flatten, inplace=inplace)


def test_fork_identity_grows_and_frees():
    rng = np.random.default_rng(4)
    say("[fork] every row goes on; every row ends")
    run_fork(fork_state(rng, 20, 30, 800, 100), np.arange(20), 64)
    op = run_fork(fork_state(rng, 20, 30, 800, 100), np.full(20, -1), 64)
    assert (op.block_table == -1).all() and (op.seq_lens == 0).all()


@pytest.mark.parametrize("spare", [0, 1, 3, 9])
def test_fork_without_pages_enough(spare):
    rng = np.random.default_rng(5)
    say(f"[fork] {spare} free pages")
    op = run_fork(fork_state(rng, 6, 20, 300, spare), [0, 0, 1, 1, 2, 2, 3, 3, 4, 5], 64)
    assert op.missing.item() > 0


def test_fork_tails_of_other_owners():
    """A partly filled page that two rows name, or that another owner holds, is copied for every child."""
    rng = np.random.default_rng(6)
    table, seq, refs, pool = fork_state(rng, 4, 10, 250, 40, share=0)
    seq[:] = [70, 70, 45, 100]
    table[:, :] = -1
    table[0, :3], table[1, :3], table[2, :2], table[3, :4] = [1, 2, 3], [1, 2, 3], [4, 5], [6, 7, 8, 9]
    refs[:] = 0
    refs[[1, 2, 3]], refs[[4, 5]], refs[[6, 7, 8, 9]] = 2, 1, 1
    refs[5] = 2
    say("[fork] shared tails")
    run_fork((table, seq, refs, pool), [0, 1, 1, 2, 3, 3], 0)


def test_fork_bad_entries_and_lengths():
    rng = np.random.default_rng(7)
    table, seq, refs, pool = fork_state(rng, 8, 12, 380, 60)
    table[0, 0], table[1, 1] = len(refs), -5
    seq[2], seq[3] = -4, 10 ** 6                              # past the table: as long as the table
    table[4, -1] = -1
    say("[fork] bad entries")
    run_fork((table, seq, refs, pool), [0, 1, 2, 3, 4, 5, 6, 7, 0, 1, 3, -9, 2 ** 31 - 1], 33)


@pytest.mark.parametrize("pages", [2047, 2048, 2049, 9000])
def test_fork_over_many_chunks(pages):
    rng = np.random.default_rng(pages)
    rows, width = 30, 40
    seq = rng.integers(1, width * 4 - 8, rows)
    need = [-(-int(n) // 4) for n in seq]
    order = rng.permutation(pages)
    table, at = np.full((rows, width), -1, np.int64), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    refs = np.bincount(table[table >= 0], minlength=pages)
    other = rng.random(pages) < 0.9
    refs[other & (refs == 0)] = 1
    say(f"[fork] {pages} pages")
    run_fork((table, seq, refs, layered_pool(rng, pages, 1, 4, 64, 0)), rng.integers(0, rows, 45), 7, page_size=4, layers=1)


# ------------------------------------------------------------ compaction

def plain_compact(host, used, table, refs):
    pages, out = len(refs), host.copy()
    live = sum(r > 0 for r in refs)
    movers = [p for p in range(live, pages) if refs[p] > 0]
    holes = [p for p in range(live) if refs[p] <= 0]
    moved = [p if refs[p] > 0 and p < live else -1 for p in range(pages)]
    counts = [refs[p] if refs[p] > 0 and p < live else 0 for p in range(pages)]
    for p, q in zip(movers, holes):
        moved[p], counts[q] = q, refs[p]
        out[q, :used] = host[p, :used]
    new = [[moved[p] if 0 <= p < pages else -1 for p in row] for row in table]
    return new, counts, moved, live, out


def run_compact(rng, pages, share, rows=7, width=31, layers=2, gap=4096, inplace=False, flatten=False):
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedPageCompact
    refs = np.where(rng.random(pages) < share, rng.integers(1, 4, pages), 0)
    table = rng.integers(-2, pages + 2, (rows, width))
    host, flat, views = layered_pool(rng, pages, layers, 4, 64, gap)
    t, r = ints(table), ints(refs)
    caches, used = ([flat], flat.shape[1]) if flatten else (views, layers * 4 * 64)
    op = PreparedPageCompact(caches, t, r, output=(t, r) if inplace else None)
    op.run()
    torch.cuda.synchronize()
    want = plain_compact(host, used, table.tolist(), refs.tolist())
    for got, expect in zip((op.block_table, op.refs, op.moved, op.live), want):
        np.testing.assert_array_equal(got.cpu().numpy().ravel(), np.asarray(expect).ravel())
    np.testing.assert_array_equal(flat.cpu().numpy(), want[4])


@pytest.mark.parametrize("pages", [1, 2, 40, 2047, 2048, 2049, 6144, 10001, 20001])
@pytest.mark.parametrize("share", [0.0, 0.05, 0.5, 0.97, 1.0])
def test_compact(pages, share):
    say(f"[compact] {pages} pages, {share} in use")
    run_compact(np.random.default_rng(pages), pages, share)


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("flatten", [False, True])
def test_compact_in_place_and_flat_backing(inplace, flatten):
    say(f"[compact] in place {inplace}, flat {flatten}")
    for pages in (1500, 3001, 17000):
        run_compact(np.random.default_rng(1), pages, 0.4, rows=100, width=77, inplace=inplace, flatten=flatten)


def test_compact_pages_of_many_slices():
    say("[compact] pages of 622592 bytes")
    run_compact(np.random.default_rng(2), 60, 0.5, layers=38 * 64, gap=16)


# ------------------------------------------------------------ offsets, graphs, streams

def test_offsets_past_32_bits():
    """A pool of 4.5 GB: pages beyond 4 GiB are copied from and to."""
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedPageCompact, PreparedPageFork, PreparedPathCommit
    pages, stride = 7300, 622592
    flat = torch.empty((pages, stride), dtype=torch.int8, device="cuda")
    flat[0].fill_(1), flat[1].fill_(2), flat[pages - 2].fill_(3), flat[pages - 1].fill_(4)
    refs = torch.ones(pages, dtype=torch.int32, device="cuda")
    refs[1] = refs[pages - 1] = 0
    say("[pages] fork past 4 GiB")
    op = PreparedPageFork(flat, ints([[pages - 2]]), ints([5]), refs, ints([0, 0, 0]))
    op.run()
    assert op.block_table.cpu().tolist() == [[pages - 2], [1], [pages - 1]]
    assert (flat[1] == 3).all() and (flat[pages - 1] == 3).all()
    refs[1], refs[pages - 2:] = 0, ints([0, 1])
    flat[pages - 1].fill_(9)
    say("[pages] compact past 4 GiB")
    op = PreparedPageCompact(flat, ints([[pages - 1, 0]]), refs)
    op.run()
    assert op.block_table.cpu().tolist() == [[1, 0]] and (flat[1] == 9).all() and op.live.item() == pages - 2
    view = flat.view(-1).as_strided((pages, 32, 512), (stride, 512, 1))
    view[pages - 1, 7].fill_(11)
    say("[pages] commit past 4 GiB")
    PreparedPathCommit(view, ints([[pages - 1]]), ints([0, 5]), ints([8]), ints([[4]]), ints([1])).run()
    assert (view[pages - 1, 3] == 11).all() and (view[pages - 1, 7] == 11).all()


def test_captured_operators_replay():
    """Fork, commit and compaction in one graph, in place, replayed over changing states, with eager work between."""
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedPageCompact, PreparedPageFork, PreparedPathCommit
    rng = np.random.default_rng(9)
    rows, width, layers = 6, 14, 2
    table, seq, refs, (host, flat, views) = fork_state(rng, rows, width, 300, 120, layers=layers)
    t, s, r, parents = ints(table), ints(seq), ints(refs), ints([0, 0, 1, 2, 2, -1])
    cu, lens, paths = ints(np.arange(rows + 1) * 9), ints([2] * rows), ints([[1, 4]] * rows)
    total = torch.empty_like(s)
    fork = PreparedPageFork(views, t, s, r, parents, room=9, output=(t, s, r))
    commit = PreparedPathCommit(views, t, cu, total, paths, lens)
    compact = PreparedPageCompact(views, t, r, output=(t, r))

    def step():
        fork.run()
        torch.add(s, 9, out=total)
        commit.run()
        s.copy_(commit.seq_lens)
        compact.run()

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    state = (table.tolist(), seq.tolist(), refs.tolist(), host)
    used = layers * BLOCK * 64
    for k in range(4):
        chosen = rng.integers(-1, rows, rows).tolist()
        nodes = sorted(rng.choice(9, 2, replace=False).tolist())
        parents.copy_(ints(chosen))
        paths.copy_(ints([nodes] * rows))
        say(f"[pages] replay {k}")
        graph.replay()
        flat.sum().item()                                   # the program's own work between
        torch.cuda.synchronize()
        new, lengths, counts, missing, data = plain_fork(state[3], used, *state[:3], chosen, 9, BLOCK)
        assert missing == 0
        data, lengths = plain_commit(data, layers, BLOCK, 64, new, list(range(0, 9 * rows + 1, 9)),
                                     [n + 9 for n in lengths], [nodes] * rows, [2] * rows)
        new, counts, _, _, data = plain_compact(data, used, new, counts)
        state = (new, lengths, counts, data)
        np.testing.assert_array_equal(t.cpu().numpy(), new)
        np.testing.assert_array_equal(s.cpu().numpy(), lengths)
        np.testing.assert_array_equal(r.cpu().numpy(), counts)
        np.testing.assert_array_equal(flat.cpu().numpy(), data)


def test_another_stream():
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedPageFork
    rng = np.random.default_rng(10)
    table, seq, refs, (host, flat, views) = fork_state(rng, 9, 12, 300, 40)
    parents = [0, 0, 1, 5, 5, 5, 8]
    op = PreparedPageFork(views, ints(table), ints(seq), ints(refs), ints(parents), room=3)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(3):                                  # a pass leaves its workspace as it was
            op.run()
    side.synchronize()
    want = plain_fork(host, 2 * BLOCK * 64, table.tolist(), seq.tolist(), refs.tolist(), parents, 3, BLOCK)
    np.testing.assert_array_equal(op.block_table.cpu().numpy(), want[0])
    np.testing.assert_array_equal(op.refs.cpu().numpy(), want[2])
    np.testing.assert_array_equal(flat.cpu().numpy(), want[4])


def test_refusals():
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedPageCompact, PreparedPageFork, PreparedPathCommit
    cache = torch.zeros((9, 32, 1, 512), dtype=torch.int8, device="cuda")
    table, seq, refs, parents = ints([[0, 1], [2, -1]]), ints([40, 3]), ints([1] * 9), ints([0, 1, 1])
    cu, paths, lens = ints([0, 3, 5]), ints([[0, 2], [1, -1]]), ints([2, 1])

    def refuse(match, make):
        with pytest.raises(ValueError, match=match):
            make()

    refuse("GPU caches", lambda: PreparedPathCommit([], table, cu, seq, paths, lens))
    refuse("GPU caches", lambda: PreparedPathCommit(cache.cpu(), table, cu, seq, paths, lens))
    refuse("same pages", lambda: PreparedPathCommit([cache, cache[:5]], table, cu, seq, paths, lens))
    refuse("16-byte", lambda: PreparedPathCommit(cache[..., :500], table, cu, seq, paths, lens))
    refuse("16-byte", lambda: PreparedPathCommit(cache.view(-1)[8:-504].view(-1, 1, 512), table, cu, seq, paths, lens))
    refuse("contiguous", lambda: PreparedPathCommit(cache.transpose(1, 3), table, cu, seq, paths, lens))
    refuse("overlap", lambda: PreparedPathCommit(cache.as_strided((9, 32, 512), (512, 512, 1)), table, cu, seq, paths, lens))
    refuse("not overlap", lambda: PreparedPathCommit([cache, cache], table, cu, seq, paths, lens))
    refuse("cu_q", lambda: PreparedPathCommit(cache, table, cu[:2], seq, paths, lens))
    refuse("INT32", lambda: PreparedPathCommit(cache, table, cu, seq.long(), paths, lens))
    refuse("block_table", lambda: PreparedPathCommit(cache, table[:1], cu, seq, paths, lens))
    refuse("path_lens", lambda: PreparedPathCommit(cache, table, cu, seq, paths, lens[:1]))
    refuse("one request", lambda: PreparedPathCommit(cache, table, cu, seq, paths[:, :0].contiguous(), lens))
    refuse("buffer of their own", lambda: PreparedPathCommit(cache, table, cu, seq, paths, lens, output=seq))

    refuse("refs", lambda: PreparedPageFork(cache, table, seq, refs[:8], parents))
    refuse("seq_lens", lambda: PreparedPageFork(cache, table, seq[:1], refs, parents))
    refuse("INT32", lambda: PreparedPageFork(cache, table, seq, refs, parents.float()))
    refuse("room", lambda: PreparedPageFork(cache, table, seq, refs, parents, room=-1))
    refuse("room", lambda: PreparedPageFork(cache, table, seq, refs, parents, room=2.0))
    refuse("pages of", lambda: PreparedPageFork(cache, table, seq, refs, parents, page_size=0))
    refuse("one row", lambda: PreparedPageFork(cache, table, seq, refs, parents[:0]))
    refuse("new block table", lambda: PreparedPageFork(cache, table, seq, refs, parents, output=(table, None, None)))
    refuse("overlap", lambda: PreparedPageFork(cache, table, seq, refs, parents, output=(None, parents, None)))
    both = ints([1] * 13)
    refuse("overlap", lambda: PreparedPageFork(cache, table, seq, both[:9], parents, output=(None, None, both[4:])))
    refuse("contiguous", lambda: PreparedPageFork(cache[:, :, :, ::2], table, seq, refs, parents))

    refuse("refs", lambda: PreparedPageCompact(cache, table, refs.long()))
    refuse("block_table", lambda: PreparedPageCompact(cache, table[0], refs))
    refuse("one row", lambda: PreparedPageCompact(cache, table[:, :0].contiguous(), refs))
    refuse("overlap", lambda: PreparedPageCompact(cache, table, both[:9], output=(None, both[1:10])))
