"""Few rows per KV head over a paged cache, in the shapes that take one way of sharing the work out or the other by a part of its own: two rounds
of chunks, column groups on the line, a context that is longer than its shares."""
import pytest
import torch

import paged_ref as ref
from test_gpu_paged import DEV, check_attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("D,most", [(64, 640), (128, 300)])
def test_two_rounds_of_chunks(kerns, D, most, eight):
    """64 sequences on 8 KV heads: more pairs than units, twice as many at most, over a table without room for long contexts."""
    c = ref.Paged([(1, (53 * i) % most) for i in range(64)], 16, 8, D, torch.float16, DEV, eight=eight)
    here = check_attend(kerns, c, 16)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):   # where a kernel of its own merges
        there = check_attend(kerns, c, 16)
    side.synchronize()
    assert torch.equal(here, there)


@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
def test_two_rounds_of_chunks_of_drafts(kerns, eight):
    c = ref.Paged([(1 + i % 3, (91 * i) % 600) for i in range(60)], 32, 6, 64, torch.bfloat16, DEV, eight=eight)
    check_attend(kerns, c, 18)


@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("Hq,Hkv,D", [(48, 1, 64), (40, 2, 64), (34, 2, 128)])
def test_line_of_column_groups(kerns, Hq, Hkv, D, eight):
    """More than 16 query heads to a KV head, and more sequences than chunks are made for."""
    c = ref.Paged([(1, (71 * i) % 500) for i in range(70)], 16, Hkv, D, torch.float16, DEV, eight=eight)
    check_attend(kerns, c, Hq)


@pytest.mark.parametrize("eight", [False, True], ids=["16", "e4m3"])
@pytest.mark.parametrize("n,Hq,Hkv", [(1, 4, 1), (2, 8, 1), (1, 20, 1)], ids=["one token", "drafts", "column groups"])
def test_line_with_one_long_context(kerns, n, Hq, Hkv, eight):
    """Short sequences and one whose rows alone set the share: as many parts as a row may have."""
    seqs = [(n, (13 * i) % 40) for i in range(66)]
    seqs[30] = (n, 31000)
    c = ref.Paged(seqs, 64, Hkv, 64, torch.float16, DEV, eight=eight)
    check_attend(kerns, c, Hq)
