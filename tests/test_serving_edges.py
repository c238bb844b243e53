"""Calls of the serving operators at the edge of what they take, as far as they can be told without a GPU."""

import os
import shutil
import subprocess

import pytest

from strassen_tpu_amd import _lib
from test_serving_surface import P, _attention, _cache, _heads

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a host compiler")
def test_overlap_of_strided_operands(tmp_path):
    exe = tmp_path / "overlap_check"
    build = subprocess.run(["g++", "-O2", "-std=c++17", "-o", str(exe), os.path.join(HERE, "overlap_check.cpp")],
                           capture_output=True, text=True, timeout=600)
    assert build.returncode == 0, build.stderr[-3000:]
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=600)
    assert run.returncode == 0 and run.stdout.startswith("ok"), run.stdout[-2000:]


Q, OUT, FAR = 1 << 30, 1 << 31, 1 << 32  # aligned addresses that no refused call reads


def _message(rc):
    return (rc, _lib.last_error())


@pytest.mark.parametrize("q,out,cache,message", [
    # every token's row over its neighbours', by a stride of zero, of one head less, of less than a head
    (_heads(data=Q), _heads(data=OUT, token=0), {}, "on each other"),
    (_heads(data=Q), _heads(data=OUT, token=7 * 128), {}, "on each other"),
    (_heads(data=Q), _heads(data=OUT, token=8 * 64, head=64), {}, "on each other"),
    # the queries one token, one head and one chunk further, or with strides of their own
    (_heads(data=Q), _heads(data=Q + 2 * 1024), {}, "queries"),
    (_heads(data=Q + 2 * 1024), _heads(data=Q), {}, "queries"),
    (_heads(data=Q), _heads(data=Q + 2 * 128), {}, "queries"),
    (_heads(data=Q), _heads(data=Q + 16), {}, "queries"),
    (_heads(data=Q), _heads(data=Q, token=2048), {}, "queries"),
    (_heads(data=Q, token=0), _heads(data=Q), {}, "queries"),
    # the cache
    (_heads(data=Q), _heads(data=OUT), {"k": OUT}, "cache"),
    (_heads(data=Q), _heads(data=OUT), {"v": OUT - 2 * 16 * 2 * 128 * 7}, "cache"),
    (_heads(data=OUT), _heads(data=OUT), {"v": OUT}, "cache"),
])
def test_attention_refuses_results_that_overlap(q, out, cache, message):
    rc, said = _message(_attention(q=q, out=out, cache=_cache(**{"k": FAR, "v": FAR + (1 << 24), **cache})))
    assert rc == _lib.SMX_ERR_INVALID and message in said, said


@pytest.mark.parametrize("q,out", [
    (_heads(data=Q), _heads(data=Q)),  # in place
    (_heads(data=Q, token=4096), _heads(data=Q + 2 * 2048, token=4096)),  # columns of one tensor
    (_heads(data=Q), _heads(data=Q + 2 * 8 * 1024)),  # behind each other
    (_heads(data=Q, token=128, head=1024), _heads(data=Q + 2 * 8 * 1024, token=128, head=1024)),
])
def test_attention_takes_results_beside_the_queries(q, out):
    """Refused for the workspace or, without a GPU, for the device, not for what they overlap."""
    rc, said = _message(_attention(q=q, out=out, cache=_cache(k=FAR, v=FAR + (1 << 24)), workspace=P))
    assert rc != _lib.SMX_OK and not any(x in said for x in ("queries", "each other", "share")), said
