"""The rotating append without a GPU: the PyTorch path against 64 bits and against rope then
kv_write, its refusals."""

from __future__ import annotations

import pytest
import torch

from mini_vllm import torch_path
from mini_vllm.kernels import extension, ops
from rope_write_helpers import append_case, clone_pools, rotated64


def call(c, pools, **more):
    args = {**c, **pools, **more}
    return ops.rope_kv_write(**args)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_rotation_and_places(dtype):
    c, pools = append_case([(5, 20), (0, 1), (40, 3)], dtype=dtype, hq=4, hk=2, d=32, padded=2)
    before = clone_pools(pools)
    q = call(c, pools)
    half = torch.finfo(dtype).eps / 2
    for got, x in ((q, c["q"]), (pools["key_pool"].view(-1, 2, 32)[c["slot_mapping"].long()], c["k"])):
        want, size = rotated64(x, c)
        # two products and a sum in float32, then the type's rounding
        bound = size * 3 * 2.0**-24 + half * (want.abs() + size * 2.0**-22) + 2.0**-25
        n = x.shape[0] - (0 if got is q else 2)  # (a padding row is not in the pool)
        assert ((got.double() - want).abs() <= bound)[:n].all()
    live = c["slot_mapping"][:-2].long()
    assert torch.equal(pools["value_pool"].view(-1, 2, 32)[live], c["v"][:-2])
    rest = torch.ones(pools["key_pool"].view(-1, 2, 32).shape[0], dtype=torch.bool)
    rest[live] = False
    for name in ("key_pool", "value_pool"):
        assert torch.equal(pools[name].view(-1, 2, 32)[rest], before[name].view(-1, 2, 32)[rest])


def test_same_type_pools_are_rope_then_kv_write():
    c, pools = append_case([(5, 20), (40, 3)], dtype=torch.bfloat16, hq=4, hk=2, d=32)
    other = clone_pools(pools)
    q = call(c, pools)
    k = torch_path.apply_rope(c["k"], c["positions"], c["cos"], c["sin"])
    torch_path.kv_write(other["key_pool"], other["value_pool"], k, c["v"], c["slot_mapping"])
    assert torch.equal(pools["key_pool"], other["key_pool"])
    assert torch.equal(pools["value_pool"], other["value_pool"])
    assert torch.equal(q, torch_path.apply_rope(c["q"], c["positions"], c["cos"], c["sin"]))


def test_fp8_values_are_within_half_a_step():
    c, pools = append_case([(5, 20), (0, 1), (40, 3)], dtype=torch.bfloat16,
                           kv_dtype=torch.float8_e4m3fn, hq=4, hk=2, d=32)
    call(c, pools)
    pages = c["slot_mapping"].long() // 16
    for name, x in (("key_pool", rotated64(c["k"], c)[0]), ("value_pool", c["v"].double())):
        scale = pools[name[0] + "_scale"][pages].double()[..., None]
        got = pools[name].view(-1, 2, 32)[c["slot_mapping"].long()].double() * scale
        # half a step of e4m3, a subnormal step's half below 2^-6, and the float32 rotation's error
        assert ((got - x).abs() <= x.abs() * 2.0**-4 * (1 + 2.0**-20) + scale * 2.0**-10).all()
        assert torch.equal(torch.log2(scale), torch.log2(scale).round())


def test_a_value_that_is_not_finite_harms_only_itself():
    def run(spoil):
        c, pools = append_case([(5, 20)], dtype=torch.float32, kv_dtype=torch.float8_e4m3fn, hq=2,
                               hk=2, d=32)
        if spoil:
            c["v"][3, 1, 7], c["v"][4, 0, 9], c["v"][5, 0, 0] = float("inf"), float("nan"), float("-inf")
        else:
            c["v"][3, 1, 7] = c["v"][4, 0, 9] = c["v"][5, 0, 0] = 0.0
        call(c, pools)
        return c, pools
    c, spoilt = run(True)
    _, clean = run(False)
    assert torch.equal(spoilt["v_scale"], clean["v_scale"])
    a, b = (x["value_pool"].view(-1, 2, 32)[c["slot_mapping"].long()].float() for x in (spoilt, clean))
    assert a[3, 1, 7] == 448 and a[5, 0, 0] == -448 and a[4, 0, 9].isnan()
    a[3, 1, 7] = a[4, 0, 9] = a[5, 0, 0] = 0.0
    assert torch.equal(a, b)


def test_strict_mode_and_refusals():
    c, pools = append_case([(5, 20)], dtype=torch.float32, hq=2, hk=2, d=32)
    with ops.strict_kernels(), pytest.raises(RuntimeError, match="device tensors"):
        call(c, pools, use_cuda=True)
    lib = extension.HipExtension(extension.open_library())
    with pytest.raises(RuntimeError, match="CUDA device"):
        lib.rope_kv_write(c["q"], c["k"], c["v"], c["positions"], c["cos"], c["sin"],
                          pools["key_pool"], pools["value_pool"], c["slot_mapping"])


def raw(lib, **more):
    """The C entry with sizes only: every refusal below comes before a pointer is looked at."""
    a = dict(positions_bytes=8, max_positions=64, tokens=4, hq=4, hk=2, d=128, block=16, blocks=8,
             dtype=2, pool=2, k_scales=None, q_stride=0, pointer=None)
    a.update(more)
    s, p = a["k_scales"], a["pointer"]
    rc = lib.mvllm_rope_kv_write(p, p, p, s, s, p, p, p, a["q_stride"], 0, 0, p, a["positions_bytes"],
                                 p, p, a["max_positions"], p, a["tokens"], a["hq"], a["hk"], a["d"],
                                 a["block"], a["blocks"], a["dtype"], a["pool"], None)
    return rc, lib.mvllm_last_error().decode()


def test_refusals_of_the_c_entry():
    lib = extension.open_library()
    for more, words in (({"block": 12}, "power of two"), ({"tokens": -1}, "bad shape"),
                        ({"blocks": 0}, "bad shape"), ({"positions_bytes": 2}, "int32 or int64"),
                        ({"d": 24}, "not served"), ({"d": 2048}, "not served"), ({"dtype": 3}, "not served"),
                        ({"dtype": 2, "pool": 1}, "not served"), ({"pool": 3, "d": 96}, "not served"),
                        ({"pool": 3}, "required for a float8 pool"), ({"k_scales": 256}, "only for one"),
                        ({}, "NULL"), ({"pointer": 8}, "16-byte aligned"),
                        ({"pointer": 256, "q_stride": 100}, "cover the token's heads"),
                        ({"pointer": 256, "q_stride": 516}, "16-byte aligned")):
        rc, message = raw(lib, **more)
        assert rc != 0 and words in message, (more, message)
    assert raw(lib, tokens=0)[0] == 0
