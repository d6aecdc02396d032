"""Sizes within each limit that are together more than a launch has: refused on the host, by the query for a workspace too, before anything is planned for them."""
import ctypes as C

import pytest

from metalhlo_amd import _lib
from tests.test_serving_host import BF16, F16, F32, I32, P, attend, cache, seqs


def _need(c, s, heads):
    return _lib.load().mhip_paged_attention_workspace(C.byref(c), C.byref(s), heads)


MANY = dict(sequences=65536, width=1, tokens=1 << 24)


@pytest.mark.timeout(60)
@pytest.mark.parametrize("c,s,heads", [(dict(heads=1024), MANY, 4096), (dict(heads=1024), MANY, 1 << 15), (dict(heads=1), MANY, 63), (dict(heads=2), dict(sequences=1, width=1, tokens=1 << 24), 126),
                                       (dict(heads=1024, head_size=128), dict(sequences=1, width=1 << 10, tokens=1 << 24), 1024),
                                       (dict(heads=2), dict(tokens=1 << 24), 1 << 41)], ids=str)
def test_more_tiles_than_a_launch_has(c, s, heads):
    c, s = cache(**c), seqs(**s)
    if heads < 1000:                                           # (fits: the query answers, and nothing is called)
        assert 0 < _need(c, s, heads) < 1 << 33
        return
    assert _need(c, s, heads) == 0
    assert attend(c, s, heads=heads) == 2, _lib.load().mhip_last_error()


@pytest.mark.timeout(60)
@pytest.mark.parametrize("c,s", [(dict(pages=1 << 62, heads=4), {}), (dict(page_size=1 << 40), {}), (dict(head_size=1 << 40), {}), ({}, dict(tokens=1 << 40)), ({}, dict(width=1 << 40)),
                                 ({}, dict(sequences=1 << 40)), (dict(heads=1 << 40), {}), (dict(head_size=48), {}), (dict(page_size=0), {}), (dict(page_size=-16), {}), ({}, dict(width=-1))], ids=str)
def test_no_workspace_for_what_is_refused(c, s):
    c, s = cache(**c), seqs(**s)
    assert _need(c, s, max(c.heads, 1) * 2) == 0
    assert attend(c, s, heads=max(c.heads, 1) * 2) in (1, 2)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows", [1 << 24, (1 << 24) + 1, 1 << 40])
def test_more_rows_of_logits_than_a_launch_has_threads_for(rows, dtype):
    code = _lib.load().mhip_token_log_probs(None, P, P, P, P, None, None, rows, 100, 0, dtype, I32, None, 0)
    assert code == 2 and b"launch" in _lib.load().mhip_last_error()
