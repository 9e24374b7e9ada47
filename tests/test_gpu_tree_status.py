"""The status word of the tree attention's bounded waits: who looks at it, and when.  (No wait is made to run out here: the word
is set by hand.)"""
import pytest
import torch

from lrqk_b200 import DynamicLRQKCache, check_tree_status, tree_attention
from lrqk_b200 import tree as tree_module
from lrqk_b200._lib import ETIMEOUT, LrqkError
from test_gpu_tree import check, make

pytestmark = pytest.mark.gpu


def _word():
    q, ck, cv, tk, tv, _ = make(1, 2, 1, 1, 3, 9, 64, torch.bfloat16)
    tree_attention(q, ck, cv, tk, tv)
    return tree_module._status[torch.cuda.current_device()]


def test_the_cache_reports_it_where_it_reports_the_others():
    word = _word()
    g = torch.Generator(device="cuda").manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()  # noqa: E731
    for how in ("check_status", "close"):
        cache = DynamicLRQKCache(r=16, num_active_tokens=64, lite_tokens=8, max_sequence_length=512, num_key_value_groups=2, init_aq_ak_method="top")
        cache.update(r(1, 4, 100, 64), r(1, 2, 100, 64), r(1, 2, 100, 64), 0)
        with cache.drafting():
            cache.attend_tree(r(1, 4, 3, 64), r(1, 2, 3, 64), r(1, 2, 3, 64), 0)
        cache.check_status()
        word[0] = ETIMEOUT
        with pytest.raises(LrqkError):
            getattr(cache, how)()
        cache.check_status()                                       # looked at once
        cache.close()


def test_a_look_waits_for_calls_on_other_streams():
    word = _word()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)                             # some 50 ms of work ahead of the failing call
        word.fill_(ETIMEOUT)
    with pytest.raises(LrqkError):
        check_tree_status()
    q, ck, cv, tk, tv, _ = make(1, 2, 1, 1, 3, 9, 64, torch.bfloat16)
    with torch.cuda.stream(side):                                  # and what it cleared is cleared for every stream
        got = tree_attention(q, ck, cv, tk, tv, return_lse=True)
    torch.cuda.synchronize()
    check(got, q, ck, cv, tk, tv)
    check_tree_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_first_call_under_capture_has_a_word_of_its_own(dtype, monkeypatch):
    q, ck, cv, tk, tv, mask = make(2, 8, 2, 2, 9, 700, 128, dtype)
    tree_attention(q, ck, cv, tk, tv, mask)                        # (libraries and streams are up; the word is hidden next)
    monkeypatch.setattr(tree_module, "_status", {})
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = tree_attention(q, ck, cv, tk, tv, mask, return_lse=True)
    assert not tree_module._status
    for _ in range(3):
        got[0].fill_(1.0)
        graph.replay()
        check(got, q, ck, cv, tk, tv, mask)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_entry_without_a_status_word_clears_its_own(dtype):
    import ctypes as C
    from lrqk_b200 import _lib
    q, ck, cv, tk, tv, _ = make(1, 8, 2, 2, 5, 900, 64, dtype)
    out, lse = torch.empty_like(q), torch.empty(1, 8, 5, device="cuda")
    a = _lib.TreeArgs(_lib.LRQK_F32 if dtype is torch.float32 else _lib.LRQK_BF16, 1, 5, 8, 2, 2, 64, 0.125, 900, q.data_ptr(), ck.data_ptr(), cv.data_ptr(),
                      tk.data_ptr(), tv.data_ptr(), *q.stride()[:3], *ck.stride()[:3], *cv.stride()[:3], *tk.stride()[:3], *tv.stride()[:3], None, None, 0,
                      out.data_ptr(), lse.data_ptr(), None)
    lib = _lib.lib()
    bytes_ = lib.lrqk_tree_attention_workspace_bytes(C.byref(a))
    ws = torch.full((bytes_ + 64,), 0xFF, dtype=torch.uint8, device="cuda")           # never initialised
    _lib.check(lib.lrqk_tree_attention(C.byref(a), ws.data_ptr(), torch.cuda.current_stream().cuda_stream), "lrqk_tree_attention")
    check((out, lse), q, ck, cv, tk, tv)
    assert ws[bytes_ - 4:bytes_].tolist() == [0] * 4 and bool((ws[bytes_:] == 0xFF).all())   # its word: cleared, the last of the workspace
