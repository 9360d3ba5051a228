"""The experts' product with the tiles that prompts take (128 x 128 and 256 x 256), against the definition in 64
bits and against the same rows in small batches."""
import pytest
import torch

import expert_ops as ops

pytestmark = pytest.mark.gpu

# (tokens, top_k, experts, weight rows) that take tiles of 128 x 128 and of 256 x 256
MIDDLE, LARGE = (1500, 2, 3, 4096), (3000, 3, 4, 4096)
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def make(cuda, T, k, E, out, K, grouped=False, seed=0, offset=0):
    gen = torch.Generator(cuda).manual_seed(seed)
    codes = lambda *s: torch.randint(-127, 128, s, dtype=torch.int8, device=cuda, generator=gen)
    near_one = lambda *s: torch.rand(*s, device=cuda, generator=gen) + 0.5
    ids = torch.randint(0, E, (T, k), dtype=torch.int32, device=cuda, generator=gen)
    ids[torch.rand(T, k, device=cuda, generator=gen) < 0.05] = -1
    n = T * k if grouped else T
    return dict(codes=codes(n, K + offset)[:, offset:], scales=near_one(n) / 127,
                weight=codes(E, out, K + offset)[:, :, offset:], weight_scales=near_one(E, out) / (127 * K ** 0.5),
                groups=ops.group_experts(ids, E), grouped=grouped)


def activated(v, act):
    if act == "relu":
        return v.clamp(min=0)
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v / 2 ** 0.5))
    return v


def check(a, act=None, gated=False, bias=None, dtype=torch.float32):
    y = ops.experts_linear_int8(**a, activation=act, gated=gated, bias=bias, dtype=dtype)
    g, k = a["groups"], a["groups"].places.shape[-1]
    at = g.offsets.tolist()
    for e in range(len(at) - 1):
        places = torch.arange(at[e], at[e + 1], device=y.device)
        r = places if a["grouped"] else g.entries[at[e]:at[e + 1]].long() // k
        acc = a["codes"][r].double() @ a["weight"][e].double().t().contiguous()
        v = acc * a["scales"][r].double()[:, None] * a["weight_scales"][e].double()
        size = v.abs()
        if bias is not None:
            v, size = v + bias[e].double(), size + bias[e].double().abs()
        if gated:
            n = v.shape[1] // 2
            gate = activated(v[:, :n], act)
            size = size[:, :n] * v[:, n:].abs() + gate.abs() * size[:, n:]
            v = gate * v[:, n:]
        else:
            v = activated(v, act)
        # int32 -> fp32, two products, the bias and the activation (its slope is at most 1.13, its functions
        # within 4 ulp): at most 12 half steps of what was added up; gated both factors and their product
        bound = HALF_STEP[dtype] * v.abs() + 26 * 2.0 ** -24 * size + 1e-7
        off = (y[at[e]:at[e + 1]].double() - v).abs()
        assert (off <= bound).all(), (e, float((off / bound).max()))
    if not a["grouped"]:  # a row's bits do not go by how many there are
        few = torch.tensor([0, 1, len(g.places) // 2, len(g.places) - 1], device=y.device)
        which = torch.searchsorted(g.offsets[1:].contiguous(), g.places[few], right=True).int()
        small = ops.group_experts(torch.where(g.places[few] < 0, -1, which), len(at) - 1)
        y2 = ops.experts_linear_int8(**{**a, "codes": a["codes"][few], "scales": a["scales"][few], "groups": small},
                                     activation=act, gated=gated, bias=bias, dtype=dtype)
        held = small.places >= 0
        assert held.any() and torch.equal(y2[small.places[held].long()], y[g.places[few][held].long()])
    return y


# no whole step of 128, one, two, several, each alone and with a rest; rows that start on 16 bytes and that do not
@pytest.mark.parametrize("K,offset", [(48, 0), (128, 0), (144, 0), (256, 0), (304, 0), (656, 0), (128, 1), (256, 3),
                                      (77, 0), (717, 0)])
@pytest.mark.parametrize("shape", [MIDDLE, LARGE])
@pytest.mark.parametrize("gated", [False, True])
def test_depths(cuda, shape, K, offset, gated):
    a = make(cuda, *shape, K, seed=K, offset=offset)
    check(a, "silu" if gated else None, gated)


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [MIDDLE, LARGE])
@pytest.mark.parametrize("gated,grouped", [(False, True), (True, False)])
def test_epilogue(cuda, shape, dtype, act, gated, grouped):
    """Odd numbers of columns, with a bias and without."""
    T, k, E, out = shape
    a = make(cuda, T, k, E, out - 2 if gated else out - 1, 160, grouped, seed=1)
    b = torch.randn(a["weight_scales"].shape, device=cuda, generator=torch.Generator(cuda).manual_seed(2))
    check(a, act, gated, b.to(dtype), dtype)
    check(a, act, gated, None, dtype)


# outputs of 64 MB and more, of whole 16-byte pieces: plain and gated, and of odd rows beside them
@pytest.mark.parametrize("T,k,E,out,gated,dtype", [
    (3000, 3, 4, 4096, False, torch.bfloat16), (3000, 3, 4, 4096, False, torch.float32),
    (6000, 3, 4, 4096, True, torch.float16), (6000, 3, 4, 4096, True, torch.bfloat16),
    (3000, 3, 4, 4096, True, torch.float32), (10000, 2, 16, 1736, False, torch.bfloat16),
    (3000, 3, 4, 4095, False, torch.bfloat16), (40000, 2, 64, 528, False, torch.float16)])
def test_large_outputs(cuda, T, k, E, out, gated, dtype):
    N = out // (1 + gated)
    assert T * k * N * torch.finfo(dtype).bits // 8 >= 64 << 20
    a = make(cuda, T, k, E, out, 160, seed=3)
    check(a, "silu" if gated else "relu", gated, None, dtype)


@pytest.mark.parametrize("shape", [MIDDLE, LARGE])
@pytest.mark.parametrize("gated", [False, True])
def test_large_row_scales(cuda, shape, gated):
    """Scales that alone would take the sum out of fp32, in some rows of a tile."""
    a = make(cuda, *shape, 96, seed=4)
    codes, sx, sw, w, g = (a[n] for n in ("codes", "scales", "weight_scales", "weight", "groups"))
    codes[5::50], sx[5::50] = 127, 2.0 ** 120
    sw *= 2.0 ** -110
    y = ops.experts_linear_int8(**a, gated=gated, dtype=torch.float32)
    k = g.places.shape[1]
    at = g.offsets.tolist()
    for e in range(len(at) - 1):
        r = g.entries[at[e]:at[e + 1]].long() // k
        v = (codes[r].double() @ w[e].double().t().contiguous()) * sx[r].double()[:, None] * sw[e].double()
        if gated:
            v = v[:, :v.shape[1] // 2] * v[:, v.shape[1] // 2:]
        # int32 -> fp32, two products for each factor and their product; fp32 goes down to 2^-149
        assert ((y[at[e]:at[e + 1]].double() - v).abs() <= 7 * 2.0 ** -24 * 1.01 * v.abs() + 2.0 ** -148).all()


@pytest.mark.parametrize("shape", [MIDDLE, LARGE])
def test_experts_without_rows_and_with_all(cuda, shape):
    T, k, E, out = shape
    a = make(cuda, T, k, E, out, 160, seed=5)
    for ids in (torch.zeros(T, k), torch.full((T, k), E - 1.0), (torch.arange(T * k) % 2 * (E - 1)).view(T, k)):
        check({**a, "groups": ops.group_experts(ids.to(cuda).int(), E)}, "gelu", False, None, torch.bfloat16)


@pytest.mark.parametrize("shape", [MIDDLE, LARGE])
def test_strides_of_the_weight(cuda, shape):
    a = make(cuda, *shape, 192, seed=6)
    want = check(a)
    held = int(a["groups"].offsets[-1])
    every = torch.stack([a["weight"], a["weight"] + 1], 2).flatten(1, 2)[:, ::2]  # rows apart, experts apart
    assert not every.is_contiguous()
    got = ops.experts_linear_int8(**{**a, "weight": every}, dtype=torch.float32)
    assert torch.equal(got[:held], want[:held])
