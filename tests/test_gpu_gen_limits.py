"""Generation-step operators at the ends of what they take: lengths and vocabularies, references that do not fit the table."""
from __future__ import annotations

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def jk():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import jakal_net_b200

    return jakal_net_b200


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("before", [0, 1, -1, 7])
def test_entries_without_a_reference_stay_where_they_are(jk, before):
    """Compaction of a table that names pages whose reference count is 0, past the pages in use; the workspace holds numbers
    of an earlier call, which must not be taken for pages."""
    pages = 12
    table, refs = ints([9, 10, -1], [11, 2, 40]), ints(0, 0, 1, 0, 0, 0, 0, 0, 0, 0, 1, 0)
    size = jk._LIBRARY.jk_cache_compact_workspace(pages)
    work = torch.full((size // 4,), before, dtype=torch.int32, device="cuda")
    live = ints(0)
    words = lambda *v: (ctypes.c_int64 * len(v))(*v)  # noqa: E731
    cache = words(table.data_ptr(), 3, 0, refs.data_ptr(), 2, 3, pages, 1)
    status = jk._LIBRARY.jk_cache_compact(words(0, 0, 0, 0), cache, live.data_ptr(), work.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert status == 0 and live.item() == 2
    # pages 2 and 10 are in use and go to the first two; 9 and 11 have no reference, 40 is no page
    assert table.tolist() == [[9, 1, -1], [11, 0, 40]] and refs.tolist() == [1, 1] + [0] * 10


def test_lengths_end_before_2_31(jk):
    """Tables with room for more nodes than a length can count."""
    page = 1 << 30
    most = 2 ** 31 - 65
    table, lengths, refs = ints([0, 1, -1, -1], [2, 3, -1, -1], [4, 5, -1, -1]), ints(most - 5, most - 5, 2 ** 31 - 7), ints(1, 1, 1, 1, 1, 1, 0, 0)
    added = jk.cache_reserve_([], table, lengths, refs, ints(5, 6, 100), page)
    assert added.tolist() == [5, 0, 0] and lengths.tolist() == [most, most - 5, 2 ** 31 - 7]
    assert refs.tolist() == [1] * 6 + [0, 0] and table[:, 2:].eq(-1).all()


@pytest.mark.parametrize("k", [60979, 54809, 49873, 58511])
def test_sums_over_a_large_vocabulary_keep_their_small_parts(jk, k):
    """Every entry is 1 - k 2^-42, which f32 rounds to 1 with an error of k 2^-42. With u a multiple of 2^-11 the draw lies on
    a border between two entries, and all sums up to there are exact in f64 (42 bits), as are 128 errors of 16 bits in f32: the
    token is the first entry past the border. (An f32 sum of 8192 errors rounds by up to 2^-27.)"""
    vocab = 1 << 26
    if torch.cuda.mem_get_info()[0] < 2 << 30:
        pytest.skip("needs 2 GB")
    target = torch.ones(1, 2, 1, device="cuda").expand(1, 2, vocab).contiguous()
    draft = torch.full((1, 1, vocab), k * 2.0 ** -42, device="cuda")
    tokens = torch.full((1, 1), -1, dtype=torch.int64, device="cuda")  # not accepted
    for part in (5, 77, 200, 999, 1029, 1535, 2047):
        out, accepted = jk.verify_draft(target, draft, tokens, torch.tensor([[0.5, part / 2048]], device="cuda"))
        assert accepted.tolist() == [0] and out.tolist() == [[part * (vocab // 2048), -1]]
