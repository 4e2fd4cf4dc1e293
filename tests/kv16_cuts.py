"""``attention16_cuts.cpp``, built once a session: how a call of the 16-bit cache's attention is cut."""
import ctypes
import os
import subprocess
from dataclasses import dataclass

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "qwen2-7b-triton_engine_amd", "csrc")


@dataclass
class Cuts:
    decode_items: int
    decode_grid: int
    decode_splits: int
    decode_longest: int
    decode_wrong: int
    tile_items: int
    tile_grid: int
    tile_splits: int
    tile_longest: int
    tile_wrong: int
    tile_sums: int
    parts: int
    combine: int
    limit: int
    places: int

    def check(self):
        """Every item once and with tokens, a workgroup for each and one more, places for what is joined."""
        assert self.decode_wrong == 0 and self.tile_wrong == 0, self
        assert self.decode_items <= max(0, self.decode_grid - 1) and self.tile_items <= max(0, self.tile_grid - 1), self
        assert self.tile_splits <= 1 or (self.tile_sums and self.combine), self
        assert self.decode_splits <= 1 or self.combine, self
        assert self.places >= 16 * self.decode_grid + (128 * self.tile_grid if self.tile_sums else 0), self
        return self


def build(folder) -> "callable":
    lib = os.path.join(str(folder), "libcuts16.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fPIC", "-shared", f"-I{CSRC}",
                    os.path.join(HERE, "attention16_cuts.cpp"), "-o", lib], check=True)
    fn = ctypes.CDLL(lib).attention16_cuts

    def cuts(requests, group, kvh, *, window=0, total=None, max_query=None, width=None, page=64) -> Cuts:
        """Of ``[(length, rows)]``."""
        lens = [n for n, _ in requests]
        starts = [sum(m for _, m in requests[:b]) for b in range(len(requests) + 1)]
        total = starts[-1] if total is None else total
        max_query = max(1, max(m for _, m in requests)) if max_query is None else max_query
        width = -(-max(max(lens), 1) // page) if width is None else width
        out = (ctypes.c_longlong * 15)()
        ints = lambda v: (ctypes.c_int * len(v))(*v)  # noqa: E731
        fn(len(requests), ints(starts), ints(lens), total, max_query, group, kvh, width, page.bit_length() - 1, window, out)
        return Cuts(*out)

    return cuts
