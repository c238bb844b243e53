"""Calls of the serving operators at the edge of what they take, as far as they can be told without a GPU."""

import os
import shutil
import subprocess

import pytest
import torch

import strassen_tpu_amd as smx
from strassen_tpu_amd import _lib
from test_serving_surface import P, _attention, _cache, _heads, _plan, _weight, _write

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


PAGE = 16 * 2 * 128  # elements of the test cache's page


@pytest.mark.parametrize("change,message", [
    # pages, slots and heads nearer to each other than they are long
    (dict(cache=_cache(k=Q, v=OUT, page_stride=PAGE - 128)), "each other"),
    (dict(cache=_cache(k=Q, v=OUT, slot_stride=128)), "each other"),
    (dict(cache=_cache(k=Q, v=OUT, page_stride=128, slot_stride=128)), "each other"),
    # keys and values: the same, one slot, one head, half a head apart; interleaved pages of another size
    (dict(cache=_cache(k=Q, v=Q)), "keys and values"), (dict(cache=_cache(k=Q, v=Q + 2 * 256)), "keys and values"),
    (dict(cache=_cache(k=Q + 2 * 128, v=Q)), "keys and values"), (dict(cache=_cache(k=Q, v=Q + 128)), "keys and values"),
    (dict(cache=_cache(k=Q, v=Q + 2 * (PAGE - 128), page_stride=2 * PAGE)), "keys and values"),
    # heads read from the cache, a result within it or over the heads
    (dict(k=_heads(2, data=Q, token=256)), "heads must share"), (dict(v=_heads(2, data=OUT + 512, token=256)), "heads must share"),
    (dict(q=_heads(data=Q), out=FAR), "heads must share"), (dict(q=_heads(data=FAR), out=OUT + 2 * PAGE), "q_out must share"),
    (dict(q=_heads(data=FAR), out=FAR + 2 * 1024), "q_out must be"), (dict(q=_heads(data=FAR, token=2048), out=FAR), "q_out must be"),
    (dict(q=_heads(data=FAR), k=_heads(2, data=FAR + (1 << 20)), out=FAR + (1 << 20)), "q_out must be"),
])
def test_write_refuses_overlaps(change, message):
    rc, said = _message(_write(**{"cache": _cache(k=Q, v=OUT), **change}))
    assert rc == _lib.SMX_ERR_INVALID and message in said, said


@pytest.mark.parametrize("change", [{"context": FAR}, {"fresh": FAR + 28}, {"free": FAR - 8}, {"free": FAR + 4 * 8 + 12},
                                    {"context": FAR - 4}])
def test_plan_refuses_tables_over_its_lists(change):
    lists = dict(context=Q, fresh=Q + 64, free=OUT, tables=FAR, stride=8)
    rc, said = _message(_plan(**{**lists, **change}))
    assert rc == _lib.SMX_ERR_INVALID and "block_tables" in said, said


@pytest.mark.parametrize("field", ["codes", "scales"])
def test_int4_operands_that_hold_no_tensors(field):
    w = smx.int4_weight_layout(*_weight(), group=128)
    setattr(w, field, [1, 2])
    with pytest.raises(TypeError, match=f"w.{field} must be a tensor"):
        smx.int4_matmul(torch.zeros(1, 128, dtype=torch.bfloat16), w)


def _serving_calls(lens, tables, x, w):
    yield lambda: smx.paged_plan(lens, lens, tables, page_size=16, num_pages=1, tokens=1)
    yield lambda: smx.int4_matmul(x, w)


def test_tensors_without_memory_of_their_own_are_refused():
    from torch._subclasses.fake_tensor import FakeTensorMode

    w = smx.int4_weight_layout(*_weight(), group=128)
    with FakeTensorMode():
        fake = (torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                torch.zeros(1, 128, dtype=torch.bfloat16, device="cuda"))
    for call in _serving_calls(*fake, w):
        with pytest.raises(ValueError, match="plain strided tensor"):
            call()
    real = torch.zeros(1, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="plain strided tensor"):
        smx.int4_matmul(torch._neg_view(real), w)
    with pytest.raises(ValueError, match="plain strided tensor"):
        smx.int4_matmul(real.to_sparse(), w)
    for transform in (lambda f: torch.vmap(f), lambda f: lambda x: torch.func.vjp(f, x),
                      lambda f: lambda x: torch.func.jvp(f, (x,), (x,))):
        with pytest.raises(ValueError, match="plain strided tensor|gradients"):
            transform(lambda x: smx.int4_matmul(x, w))(real[None])


def test_traced_calls_are_refused():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    lens, tables = torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    x, w = torch.zeros(1, 128, dtype=torch.bfloat16), smx.int4_weight_layout(*_weight(), group=128)
    for call in _serving_calls(lens, tables, x, w):
        with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(ValueError, match="traced"):
            call()
    for mode in ("real", "fake"):
        with pytest.raises(ValueError, match="traced"):
            make_fx(lambda x: smx.int4_matmul(x, w), tracing_mode=mode)(x)


def _headers_without_torch(build, monkeypatch, tmp_path):
    command = build.host_command
    monkeypatch.setattr(build, "host_command", lambda output: [x for x in command(output) if not x.endswith("torch/include")])


def _no_compiler(build, monkeypatch, tmp_path):
    monkeypatch.setenv("CXX", str(tmp_path / "no-such-compiler"))


@pytest.mark.parametrize("missing", [_no_compiler, _headers_without_torch])
def test_library_is_built_without_the_host_module(missing, monkeypatch, tmp_path):
    """No host compiler, or no headers of torch: the library is put in place, a host module of another build is not
    left beside it, and the build says so."""
    from strassen_tpu_amd import build

    library, module = tmp_path / "library.so", tmp_path / "_serving.so"
    library.write_text("old"), module.write_text("old")
    monkeypatch.setattr(build, "LIBRARY", str(library))
    monkeypatch.setattr(build, "HOST_MODULE", str(module))
    # the device units' part of the build, whose compiler is not what is missing
    monkeypatch.setattr(build, "_compile_unit", lambda source, workdir: (source, "", ""))
    monkeypatch.setattr(build, "verify_inline_asm_kernels", lambda text: 1)
    monkeypatch.setattr(build, "verify_kernel_scratch", lambda text, require=True: 1)
    monkeypatch.setattr(build, "link_command", lambda objects, output: ["cp", objects[0], output])
    missing(build, monkeypatch, tmp_path)
    with pytest.warns(RuntimeWarning, match="host module was not built"):
        assert build.build() == str(library)
    assert library.read_text() == open(build.SOURCES[0]).read()
    assert not module.exists() and not (tmp_path / "_serving.so.tmp").exists()


def test_attention_refuses_a_scale_that_overflows():
    """The largest scales times log2 e are infinite, and an infinity times a score of zero NaN."""
    for scale in (3e38, 2.36e38, float("inf")):
        rc, said = _message(_attention(scale=scale, q=_heads(data=Q), out=_heads(data=OUT), cache=_cache(k=FAR, v=FAR + (1 << 24))))
        assert rc == _lib.SMX_ERR_INVALID and "scale" in said, said
    rc, said = _message(_attention(scale=2.35e38, q=_heads(data=Q), out=_heads(data=OUT), cache=_cache(k=FAR, v=FAR + (1 << 24))))
    assert "scale" not in said, said
