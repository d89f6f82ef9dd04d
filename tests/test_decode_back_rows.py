"""The buffers that the 4-bit cache is read back into for a prompt's chunks grow few times over a long prompt."""
from flashbfp_b200.decode import back_rows


def _grown(chunks, cache):
    have, sizes, at = 0, [], 0
    for n in chunks:
        at += n
        room = back_rows(have, at, cache)
        assert room >= at
        if room != have:
            have = room
            sizes.append(room)
    return sizes


def test_few_growths():
    for chunk, total in ((128, 131072), (4096, 131072), (1, 5000), (1024, 1 << 20)):
        sizes = _grown([chunk] * (total // chunk), total)
        assert len(sizes) <= 12 and sizes[-1] <= total
        assert sum(sizes) <= 3 * total + 4096              # what an allocator that keeps everything holds


def test_sizes():
    assert back_rows(0, 1, 64) == 64 and back_rows(0, 100, 10000) == 1024
    assert back_rows(1024, 1000, 10000) == 1024 and back_rows(1024, 1025, 10000) == 2048
    assert back_rows(8192, 8193, 9000) == 9000 and back_rows(2048, 9000, 9000) == 9000
    assert back_rows(9000, 9100, 9000) == 9100             # positions that do not fit: the call records them
    assert back_rows(0, 0, 64) == 0
