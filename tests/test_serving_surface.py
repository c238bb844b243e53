"""The serving operators' argument checks that need no GPU: layouts of 4-bit weights on the CPU, and
refusals of the C entry points before any launch."""

import ctypes

import pytest
import torch

import strassen_tpu_amd as smx
from strassen_tpu_amd import _lib


def _weight(k=128, n=40, group=128):
    return (torch.zeros(k, n, dtype=torch.uint8), torch.ones(k // group, n, dtype=torch.bfloat16),
            torch.zeros(k // group, n, dtype=torch.uint8))


@pytest.mark.parametrize("change,message", [
    ({"codes": torch.zeros(128, 40)}, "uint8"), ({"codes": torch.full((128, 40), 16, dtype=torch.uint8)}, "0 .. 15"),
    ({"scales": torch.ones(1, 40)}, "bf16"), ({"scales": torch.ones(2, 40, dtype=torch.bfloat16)}, "scales"),
    ({"zeros": torch.full((1, 40), 16, dtype=torch.uint8)}, "0 .. 15"), ({"zeros": torch.zeros(1, 41, dtype=torch.uint8)}, "zeros"),
    ({"group": 48}, "group"), ({"group": 256}, "group"), ({"epilogue": "geglu"}, "swiglu"),
])
def test_int4_layout_refusals(change, message):
    codes, scales, zeros = _weight()
    args = {"codes": codes, "scales": scales, "zeros": zeros, "group": 128, **change}
    with pytest.raises(ValueError, match=message):
        smx.int4_weight_layout(**args)


def test_int4_layout_swiglu_needs_an_even_width():
    codes, scales, zeros = _weight(n=41)
    with pytest.raises(ValueError, match="even"):
        smx.int4_weight_layout(codes, scales, zeros, group=128, epilogue="swiglu")


@pytest.mark.parametrize("k,n,group,swiglu", [(32, 1, 32, False), (192, 40, 64, False), (256, 34, 128, True),
                                              (96, 70, 32, True)])
def test_int4_layout(k, n, group, swiglu):
    """Every word of the layout, from its description."""
    g = torch.Generator().manual_seed(k + n)
    codes = torch.randint(0, 16, (k, n), generator=g, dtype=torch.uint8)
    scales = torch.randn(k // group, n, generator=g).to(torch.bfloat16)
    zeros = torch.randint(0, 16, (k // group, n), generator=g, dtype=torch.uint8)
    w = smx.int4_weight_layout(codes, scales, zeros, group=group, epilogue="swiglu" if swiglu else None)
    half = n // 2
    tiles = 2 * -(-half // 16) if swiglu else 2 * -(-n // 32)
    assert w.codes.shape == (tiles, -(-k // 128), 4, 16, 4)
    assert w.scales.shape == (tiles, -(-k // 128), 16, 128 // group)
    words = w.codes.to(torch.int64) & 0xffffffff
    pairs = w.scales.to(torch.int64) & 0xffffffff
    for tile in range(tiles):
        for c in range(16):
            if swiglu:
                inside = tile // 2 * 16 + c
                column = inside + half * (tile % 2) if inside < half else None
            else:
                column = tile * 16 + c if tile * 16 + c < n else None
            for kk in range(-(-k // 128) * 128):
                word = int(words[tile, kk // 128, kk % 32 // 8, c, kk % 128 // 32])
                j = kk % 8
                want = int(codes[kk, column]) if column is not None and kk < k else 0
                at = 16 * (j % 2) + 4 * (j // 2) + 3
                assert (word | word << 32) >> at & 15 == want
            for gr in range(k // group):
                pair = int(pairs[tile, gr * group // 128, c, gr % (128 // group)])
                as_bf16 = lambda bits: torch.tensor([bits - (bits >> 15 << 16)], dtype=torch.int16).view(torch.bfloat16)
                if column is None:
                    assert pair == 0
                else:
                    assert as_bf16(pair >> 16)[0] == scales[gr, column]
                    assert float(as_bf16(pair & 0xffff)[0]) == -(16 + int(zeros[gr, column]))


def test_cpu_tensors_are_refused():
    lens, tables = torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="HIP device"):
        smx.paged_plan(lens, lens, tables, page_size=16, num_pages=1, tokens=1)
    w = smx.int4_weight_layout(*_weight(), group=128)
    with pytest.raises(ValueError, match="HIP device"):
        smx.int4_matmul(torch.zeros(1, 128, dtype=torch.bfloat16), w)


P = 4096  # an aligned address that no refused call reads


def _plan(**kw):
    a = dict(requests=2, width=4, page_size=16, num_pages=8, tokens=8, max_new=4, max_context=64, context=P, fresh=P,
             tables=P, stride=4, free=P, count=3, starts=P, rows=P, known=P, positions=P, slots=P, status=P, used=P)
    a.update(kw)
    return _lib.load().smx_paged_plan(*a.values(), None)


@pytest.mark.parametrize("change", [
    {"requests": 0}, {"requests": 8193}, {"tokens": 0}, {"tokens": (1 << 20) + 1}, {"page_size": 24}, {"page_size": 4},
    {"page_size": 8192}, {"width": 0}, {"num_pages": 0}, {"num_pages": 1 << 30}, {"stride": 3}, {"max_new": -1},
    {"max_context": 65}, {"max_context": -1},
    {"max_context": (1 << 30) + 1, "width": 1 << 27, "stride": 1 << 27}, {"count": -1}, {"free": None}, {"context": None}, {"slots": None}])
def test_plan_refusals(change):
    assert _plan(**change) == _lib.SMX_ERR_INVALID
    assert _lib.last_error()


def _cache(**kw):
    a = dict(k=P, v=P, page_stride=16 * 2 * 128, slot_stride=2 * 128, head_stride=128, num_pages=8, page_size=16, kv_heads=2,
             head_dim=128)
    a.update(kw)
    return _lib.SmxPagedCache(*a.values())


def _heads(heads=8, data=P, token=1024, head=128):
    return _lib.SmxHeads(data, token, head, heads)


BAD_CACHES = [{"k": None}, {"v": P + 8}, {"page_stride": 12}, {"slot_stride": 100}, {"slot_stride": 64}, {"head_stride": 8},
              {"num_pages": 0}, {"page_size": 12}, {"kv_heads": 0}, {"head_dim": 96}, {"slot_stride": 1 << 27}, {"page_stride": 1 << 31}, {"head_stride": 1 << 31},
              {"num_pages": 1 << 28}]


def _step(**kw):
    a = dict(requests=2, tokens=8, max_new=4, tables=P, stride=4, starts=P, rows=P, context=P, positions=P)
    a.update(kw)
    return _lib.SmxPagedStep(*a.values())


def _attention(cache=None, step=None, q=None, out=None, scale=0.1, window=0, workspace=P, size=0):
    return _lib.load().smx_paged_attention(cache or _cache(), step or _step(), q or _heads(), out or _heads(), scale, window, 0,
                                           workspace, size, None)


@pytest.mark.parametrize("change", [{"cache": _cache(**c)} for c in BAD_CACHES] + [
    {"step": _step(requests=0)}, {"step": _step(tokens=0)}, {"step": _step(tables=None)}, {"step": _step(positions=None)},
    {"q": _heads(7)}, {"q": _heads(258), "out": _heads(258)}, {"out": _heads(4)}, {"q": _heads(data=P + 2)}, {"q": _heads(token=1025)},
    {"out": _heads(head=130)}, {"scale": 0.0}, {"scale": float("nan")}, {"window": -1}])
def test_attention_refusals(change):
    assert _attention(**change) in (_lib.SMX_ERR_INVALID, _lib.SMX_ERR_UNSUPPORTED)
    assert _lib.last_error()


def _write(cache=None, tokens=8, q=None, k=None, v=None, cos=None, sin=None, rows=0, stride=0, q_scale=None, k_scale=None,
           dtypes=0, eps=1e-6, out=None):
    return _lib.load().smx_paged_write(cache or _cache(), tokens, P, P, q, k or _heads(2), v or _heads(2), cos, sin, rows, stride,
                                       q_scale, k_scale, dtypes, eps, out, None)


@pytest.mark.parametrize("change", [{"cache": _cache(**c)} for c in BAD_CACHES] + [
    {"tokens": 0}, {"k": _heads(3)}, {"v": _heads(2, token=3)}, {"q": _heads()}, {"out": P}, {"q": _heads(0), "out": P},
    {"q": _heads(), "out": P + 2}, {"cos": P}, {"cos": P, "sin": P, "rows": 0, "stride": 64},
    {"cos": P, "sin": P, "rows": 9, "stride": 32}, {"cos": P, "sin": P + 2, "rows": 9, "stride": 64}, {"q_scale": P}, {"k_scale": P + 4},
    {"dtypes": 8}, {"eps": -1.0}, {"eps": float("nan")}])
def test_write_refusals(change):
    assert _write(**change) in (_lib.SMX_ERR_INVALID, _lib.SMX_ERR_UNSUPPORTED)
    assert _lib.last_error()


def _int4(w=None, m=4, x=P, ldx=256, epilogue=0, extra=None, lde=0, f32=0, out=P, ldo=64):
    w = w or _lib.SmxInt4Weight(P, P, 256, 64, 128, 0, 1)
    return _lib.load().smx_int4_matmul(w, m, x, ldx, epilogue, extra, lde, f32, out, ldo, None, 0, None)


@pytest.mark.parametrize("change", [
    {"w": _lib.SmxInt4Weight(None, P, 256, 64, 128, 0, 1)}, {"w": _lib.SmxInt4Weight(P, P + 4, 256, 64, 128, 0)},
    {"w": _lib.SmxInt4Weight(P, P, 240, 64, 128, 0, 1)}, {"w": _lib.SmxInt4Weight(P, P, 256, 64, 96, 0)},
    {"w": _lib.SmxInt4Weight(P, P, 256, 64, 128, 1, 1)}, {"w": _lib.SmxInt4Weight(P, P, 256, 63, 128, 1), "epilogue": 1}, {"m": 0},
    {"x": P + 2}, {"ldx": 255}, {"ldx": 248}, {"epilogue": 1}, {"epilogue": 4}, {"epilogue": 5}, {"epilogue": 2}, {"extra": P},
    {"epilogue": 2, "extra": P, "lde": 63}, {"ldo": 63}, {"out": P + 4}, {"out": None}])
def test_int4_refusals(change):
    assert _int4(**change) in (_lib.SMX_ERR_INVALID, _lib.SMX_ERR_UNSUPPORTED)
    assert _lib.last_error()


def test_limits_match_the_header():
    import os
    import re

    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include",
                               "strassen_mi355x.h")).read()
    for name in ("SMX_PAGED_MAX_REQUESTS", "SMX_PAGED_Q_SCALE_F32", "SMX_PAGED_K_SCALE_F32", "SMX_PAGED_ROPE_F32"):
        assert int(re.search(rf"#define {name} (\d+)", header).group(1)) == getattr(_lib, name)
    for name in ("OK", "BAD_LENGTH", "OUT_OF_ROWS", "OUT_OF_PAGES", "BAD_PAGE"):
        assert int(re.search(rf"#define SMX_PAGED_{name} (\d+)", header).group(1)) == getattr(smx, f"PAGED_{name}")
    # the structures as the header lists them
    kinds = {"int64_t": ctypes.c_int64, "int32_t": ctypes.c_int32}
    for name, struct in (("paged_cache", _lib.SmxPagedCache), ("heads", _lib.SmxHeads), ("paged_step", _lib.SmxPagedStep),
                         ("int4_weight", _lib.SmxInt4Weight)):
        body = re.search(rf"typedef struct smx_{name} \{{(.*?)\}} smx_{name};", header, re.S).group(1)
        fields = []
        for line in (x.strip() for x in body.split(";")):
            if line:
                ctype, names = re.match(r"(?:const )?(\w+)\s*(.*)", line, re.S).groups()
                fields += [kinds.get(ctype, ctypes.c_void_p) if not n.strip().startswith("*") else ctypes.c_void_p
                           for n in names.split(",")]
        assert fields == [t for _, t in struct._fields_], name
