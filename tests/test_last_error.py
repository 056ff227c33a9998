"""The text of failed calls that have no handle, across threads: no GPU is needed."""
import ctypes
import threading

import gpt_oss_amd_b200 as pkg  # noqa: F401
from gpt_oss_amd_b200 import capi


def _text():
    return capi.lib().moe_b200_last_error(None)


def _elsewhere(fn):
    out = []
    t = threading.Thread(target=lambda: out.append(fn()))
    t.start()
    t.join()
    return out[0]


def _create_fails():
    h = ctypes.c_void_p()
    return capi.lib().moe_b200_create(ctypes.byref(capi.Config()), ctypes.byref(h))


def _norm_fails():
    return capi.lib().moe_b200_add_rmsnorm(None, None)


def _route_fails():
    return capi.lib().moe_b200_route_logits(None, None)


def test_a_failed_create_is_explained_in_every_thread():
    assert _elsewhere(_create_fails) == capi.ERR_INVALID
    assert b"hidden_dim" in _text() and b"hidden_dim" in _elsewhere(_text)


def test_a_failed_create_replaces_what_the_reader_failed_at_before():
    assert _norm_fails() == capi.ERR_INVALID and b"add_rmsnorm" in _text()
    assert _elsewhere(_create_fails) == capi.ERR_INVALID
    assert b"hidden_dim" in _text()
    assert _norm_fails() == capi.ERR_INVALID and b"add_rmsnorm" in _text()


def test_a_failed_operator_is_explained_in_its_thread_only():
    assert _norm_fails() == capi.ERR_INVALID
    assert b"route_logits" in _elsewhere(lambda: (_route_fails(), _text())[1])
    assert b"add_rmsnorm" in _text()


def test_many_threads_fail_at_once():
    """Each reads its own text while others fail and create handles in vain."""
    def work(fail, name):
        for _ in range(2000):
            assert fail() == capi.ERR_INVALID
            text = _text()
            if not (name in text or b"hidden_dim" in text):
                return text
        return None

    out = []
    jobs = [(_norm_fails, b"add_rmsnorm"), (_route_fails, b"route_logits"), (_create_fails, b"hidden_dim")] * 3
    threads = [threading.Thread(target=lambda j=j: out.append(work(*j))) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert out == [None] * len(jobs)
