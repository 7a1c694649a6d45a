"""How the roles of the grouped kernel (grouped_gemm.cu) take their tiles, as its source has it: a role reads a
tile from shared memory in several accesses and gives the slot back with an arrival that orders nothing, after
which the slot is written again.  So a value of every access has to be used before the arrival, by all lanes
that read (a wrong order shows on a GPU only by chance)."""
import re
from pathlib import Path

SOURCE = re.sub(r"//[^\n]*", "", (Path(__file__).resolve().parent.parent / "cumpsgemm_b200" / "csrc" /
                                  "grouped_gemm.cu").read_text())


def _body(start):
    """The braces behind `start`."""
    i = SOURCE.index("{", SOURCE.index(start))
    depth, at = 0, i
    while True:
        depth += {"{": 1, "}": -1}.get(SOURCE[at], 0)
        at += 1
        if depth == 0:
            return SOURCE[i + 1:at - 1]


def _words_of_the_reads():
    reads = re.findall(r"ld_shared_v4\(at[^,]*,([^)]*)\)", _body("void read(Tile &x) const"))
    return [re.findall(r"x\.(\w+)", r) for r in reads]


def test_a_tile_is_read_whole():
    fields = re.search(r"struct alignas\(16\) Tile \{(.*?)__device__", SOURCE, re.S).group(1)
    names = [n for line in re.findall(r"uint32_t ([^;]*);", fields) for n in re.split(r"\s*,\s*", line.strip())]
    assert sum(_words_of_the_reads(), []) == names and len(names) == 12


def test_a_slot_is_given_back_when_every_read_has_come():
    take = _body("void take(const Tile &x)")
    before = take[:take.index("mbar_arrive_cluster_relaxed")]
    for words in _words_of_the_reads():
        assert any(re.search(rf"\bx\.{w}\b", before) for w in words), words
    # all lanes of a warp read, one arrives: it waits for what the others have compared
    assert re.search(r"if \(WARP\)[^;]*__all_sync\(0xffffffffu, has_come\)", before)


def test_the_words_that_are_compared_are_never_all_ones():
    """Group numbers, blocks of K and slices of a real tile; the tile that ends the launch is all zeros."""
    take = _body("void take(const Tile &x)")
    assert set(re.findall(r"\bx\.(\w+)", take)) == {"group", "k0", "slices"}
    assert "x = Tile{};" in SOURCE
