"""Cases of attention over 4-bit pages for each kernel and each way to cut the work, with the
form that each is meant to take.  What the host is told (num_seqs, max_q, max_kv) decides
about it; the sequences that have tokens at all are few."""
import itertools
from dataclasses import dataclass

import torch

DTYPES = (torch.bfloat16, torch.float16)


@dataclass(frozen=True)
class Form:
    name: str
    rows: int            # of a block; 256 stands for the large ones, 128 rows in heads of 256 values
    wide: bool           # eight waves to a sequence
    cut: bool            # into parts, which a second launch joins
    seqs: int
    max_q: int
    max_kv: int
    ratio: int
    lens: tuple          # tokens of the sequences that have any, and their new ones
    new: tuple
    refill: dict         # heads' size -> tokens after which a wave looks up further pages

    def window(self):
        return self.lens[0] - 137 if self.refill else 2700

    def block_rows(self, d):
        return 128 if self.rows == 256 and d == 256 else self.rows


HK = 2
_FOUR = {64: 4096, 128: 4096, 256: 4096}
FORMS = (
    Form("16 rows", 16, False, False, 3, 1, 200, 4, (9000, 40, 1), (1, 1, 1), _FOUR),
    Form("16 rows, many sequences", 16, False, False, 2048, 1, 3000, 4, (4700, 33), (1, 1), _FOUR),
    Form("16 rows, eight waves", 16, True, False, 2, 1, 600, 4, (17000, 300), (1, 1), {64: 8192, 128: 8192, 256: 8192}),
    Form("16 rows, cut", 16, False, True, 3, 1, 100000, 4, (6000, 2, 700), (1, 1, 1), {}),
    Form("16 rows twice, cut", 16, False, True, 2, 6, 3000, 4, (3100, 50), (6, 3), {}),
    Form("32 rows", 32, False, False, 2048, 5, 3000, 4, (4700, 3, 40), (5, 3, 1), {64: 4096, 128: 4096, 256: 2048}),
    Form("32 rows, cut", 32, False, True, 160, 5, 6000, 4, (6000, 3, 40), (5, 3, 1), {}),
    Form("32 rows twice, cut", 32, False, True, 64, 12, 1900, 4, (1900, 3, 40), (12, 3, 7), {}),
    Form("large", 256, False, False, 2, 1500, 512, 16, (2300, 60), (20, 9), {64: 1024, 128: 1024, 256: 1024}),
    Form("large, cut", 256, False, True, 2, 300, 100000, 16, (2900, 60), (20, 9), {}))

MASKS = (("causal", True, False), ("causal, window", True, True), ("all", False, False), ("window", False, True))

CASES = tuple(itertools.product(FORMS, (64, 128, 256), MASKS, DTYPES))


def case_id(case):
    form, d, mask, dt = case
    return f"{form.name}-{d}-{mask[0]}-{str(dt)[6:]}"
