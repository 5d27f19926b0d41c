"""How the token-line kernels cut their work: the host's rules restated, so that tests can say which
paths their sizes reach.  ``test_token_line_cuts.py`` holds them against the library's workspace sizes."""

from collections import namedtuple

SIMDS, CUS = 1024, 256


def ceil(a, b):
    return -(-a // b)


def padded(states):
    return 8 if states <= 8 else 16 if states <= 16 else 32


def tiles(channels, groups, width=64):
    return ceil(channels // groups, width) * groups


def forward_chunk(batch, length, channels, groups):
    """Tokens a chunk of the scan's forward (``forward_chunk`` of ``csrc/state_space.hip``)."""
    blocks, lines = ceil(length, 16), batch * tiles(channels, groups)
    issue = (0.0, 9.5, 5.8, 5.2, 4.9, 4.5, 4.5)

    def time(per, waves):
        each = ceil(waves, SIMDS)
        return (per * 16 + 8) * each * issue[min(each, 6)] * 118 / 2300

    best, least = blocks, time(blocks, lines)
    most = ceil(blocks * lines, SIMDS) + 1
    first = ceil(most, 8)
    for per in range(first, min(most, blocks - 1, first + 255) + 1):
        chunks = ceil(blocks, per)
        t = 1.8 * time(per, chunks * lines) + 1.6e-3 * chunks * lines + 10.0
        if t < least:
            best, least = per, t
    return best * 16


Cut = namedtuple("Cut", "chunk chunks fine fine_chunks pieces")


def backward_cut(batch, length, channels, states, groups):
    """The scan's backward (``make_cut`` of ``csrc/state_space_backward.hip``): tokens a chunk of the
    gradients' pass and chunks a line, the same of the adjoints' pass, and how many of its chunks
    make one of the others."""
    wide = tiles(channels, groups, 128 if states <= 8 else 64)
    waves = 3 if states <= 8 else 4 if states <= 16 else 2
    blocks = ceil(length, 16)
    chunks = CUS * waves // (batch * wide)
    chunks = 1 if chunks < 1 or blocks <= 4 else min(chunks, blocks)
    chunk = ceil(blocks, chunks) * 16
    chunks = ceil(length, chunk)
    pieces = 1
    while (pieces < 16 and chunks > 1 and chunk // pieces >= 32
           and batch * tiles(channels, groups) * chunks * pieces * 2 <= 4096 * 5 // 4):
        pieces *= 2
    return Cut(chunk, chunks, chunk // pieces, 1 if chunks == 1 else ceil(length, chunk // pieces), pieces)


def sum_splits(rows, width):
    """Workgroups that the rows of partial parameter gradients are split over (``csrc/param_sum.hip``);
    two launches where there are several."""
    s = min(512 // ceil(width, 64), rows // 256)
    return s if s >= 2 else 1


def sum_bytes(rows, width):
    s = sum_splits(rows, width)
    return 4 * s * width if s > 1 else 0


def maps_floats(batch, length, groups, states):
    return 2 * batch * length * groups * padded(states)


def forward_bytes(batch, length, channels, states, groups):
    chunks = ceil(length, forward_chunk(batch, length, channels, groups))
    floats = maps_floats(batch, length, groups, states)
    if chunks > 1:
        floats += batch * tiles(channels, groups) * 64 * ((chunks - 1) * padded(states) + chunks)
    return 4 * floats


def backward_bytes(batch, length, channels, states, groups):
    cut, S = backward_cut(batch, length, channels, states, groups), padded(states)
    wide, columns = tiles(channels, groups, 128 if states <= 8 else 64), tiles(channels, groups) * 64
    floats = wide * batch * length * 2 * S
    floats += batch * columns * ((cut.fine_chunks - 1) * S + cut.fine_chunks + cut.chunks * (S + 2))
    floats += maps_floats(batch, length, groups, states)
    return 4 * floats + sum_bytes(batch * cut.chunks, (S + 2) * columns)
