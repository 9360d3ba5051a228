"""What each entry point of the routing refuses by itself, before any call of the device."""
import ctypes

import pytest

import rxmet_lib


@pytest.mark.parametrize("entry", ["forward", "backward"])
def test_routers(entry):
    lib = rxmet_lib.load()
    buf = (ctypes.c_float * 64)()
    p = ctypes.addressof(buf) // 16 * 16 + 16

    def route(tokens=1, dtype=0, stride=8, at=p, router=True, **kw):
        r = rxmet_lib.Router(**{**dict(experts=8, top_k=2, score=0, renormalize=1, groups=1, top_groups=1,
                                       group_best=1, scale=1.0), **kw})
        r = ctypes.byref(r) if router else None
        if entry == "forward":
            return lib.rxmet_route_forward(r, at, stride, None, p, p, tokens, dtype, None)
        return lib.rxmet_route_backward(r, at, stride, p, p, p, tokens, dtype, None)

    for kw, text in ((dict(experts=1025), "1 to 1024 experts"), (dict(experts=0), "1 to 1024 experts"),
                     (dict(score=2), "unknown score"), (dict(score=-1), "unknown score"),
                     (dict(groups=3), "equal length"), (dict(groups=0), "equal length"),
                     (dict(top_groups=2), "top_groups"), (dict(top_groups=0), "top_groups"),
                     (dict(group_best=0), "group_best"), (dict(group_best=3), "group_best"),
                     (dict(top_k=9), "top_k"), (dict(top_k=0), "top_k"), (dict(groups=4, top_k=3), "top_k"),
                     (dict(dtype=3), "fp32, fp16 or bf16"), (dict(tokens=-1), "tokens"),
                     (dict(tokens=(1 << 24) + 1), "tokens"), (dict(stride=-1), "stride"), (dict(at=None), "needed"),
                     (dict(router=False), "router is missing")):
        assert route(**kw) == -22 and text in lib.rxmet_last_error().decode(), (kw, lib.rxmet_last_error())
    assert route(tokens=0) == 0
