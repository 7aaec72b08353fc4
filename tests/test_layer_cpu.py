"""CPU tests of the layer operators' entry points: what they refuse, in which order, and the order of gated rows.  No
call here reaches a device: what is not refused by its arguments ends at the check for one."""
import ctypes

import pytest
import torch

from w4a16_opt import capi, interleave_gate_up

DEVICE = (13, 14)


@pytest.fixture(autouse=True)
def _no_device(request):
    """The addresses of these calls are not real: with a device they would be used."""
    if torch.cuda.is_available():
        pytest.skip("for machines without a GPU")


def linear(M=4, N=64, K=512, groups=8, variant=-1, flags=0, Wp=0x10000, x=0x20000, scales=0x30000, y=0x40000, words=None, **epilogue):
    lib = capi.load()
    e = capi.Epilogue(**epilogue)
    st = lib.w4a16_linear(Wp, x, scales, y, M, N, K, groups, N * K // 8 if words is None else words, ctypes.byref(e), variant, flags, None, 0,
                          None)
    return st, capi.last_error(lib)


@pytest.mark.parametrize("kw,status,msg", [
    (dict(M=0), 3, "M must be"), (dict(K=32, groups=1), 5, "multiple of 64"), (dict(N=0), 6, "at least 16"), (dict(words=1), 8, "words"),
    (dict(x=0x20008), 9, "aligned"), (dict(y=None), 1, "non-null"), (dict(activation=5), 21, "activation"),
    (dict(activation=-1), 21, "activation"), (dict(flags=8), 17, "unknown flag"), (dict(y=0x40002), 9, "4-byte"),
    (dict(bias=0x50001), 9, "aligned"), (dict(residual=0x50001), 9, "aligned"), (dict(y=0x20000), 22, "overlap"),
    (dict(y=0x20000 + 4 * 512 * 2 - 4), 22, "overlap"), (dict(y=0x10000), 22, "overlap"), (dict(y=0x30000 + 8 * 64 * 2 - 4), 22, "overlap"),
    (dict(residual=0x40000 + 64), 22, "overlap"), (dict(residual=0x40000 - 2), 22, "overlap"), (dict(bias=0x40000 + 4 * 64 * 2 - 2), 22, "overlap"),
])
def test_linear_refuses(kw, status, msg):
    st, err = linear(**kw)
    assert st == status and msg in err, (st, err)


@pytest.mark.parametrize("kw", [dict(), dict(residual=0x40000), dict(gated=1, residual=0x40000 + 4 * 32 * 2), dict(bias=0x50002, activation=4)])
def test_linear_accepts(kw):
    st, err = linear(**kw)
    assert st in DEVICE, (st, err)


def norm(**kw):
    lib = capi.load()
    args = dict(x=0x10000, weight=0x20000, y=0x30000, x_token_stride=64, y_token_stride=64, tokens=4, heads=1, dim=64, eps=1e-5)
    args.update(kw)
    a = capi.NormArgs(**args)
    st = lib.w4a16_rms_norm(ctypes.byref(a), None)
    return st, capi.last_error(lib)


RES = dict(residual=0x40000, residual_out=0x50000, residual_token_stride=64, residual_out_token_stride=64)


@pytest.mark.parametrize("kw,status,msg", [
    (dict(dim=0), 23, "dim"), (dict(dim=12), 23, "dim"), (dict(dim=32776), 23, "dim"), (dict(heads=0), 23, "heads"), (dict(heads=-1), 23, "heads"),
    (dict(dtype=2), 20, "dtype"), (dict(tokens=1 << 31), 4, "int32"), (dict(tokens=-1), 4, "int32"), (dict(tokens=1 << 62, heads=4), 4, "int32"),
    (dict(eps=-1.0), 23, "eps"), (dict(eps=float("nan")), 23, "eps"), (dict(eps=float("inf")), 23, "eps"), (dict(x=None), 1, "non-null"),
    (dict(residual=0x40000), 1, "residual_out"), (dict(x=0x10008), 9, "aligned"), (dict(x_token_stride=68), 9, "strides"),
    (dict(weight=0x20008), 9, "aligned"), (dict(x_token_stride=-64), 23, "strides"), (dict(x_token_stride=1 << 40), 23, "strides"),
    (dict(y_token_stride=0), 22, "rows of an output"), (dict(y_token_stride=56), 22, "rows of an output"),
    (dict(heads=2, y_head_stride=64, y_token_stride=64), 22, "rows of an output"), (dict(y=0x10000 + 128), 22, "very view"),
    (dict(y=0x10000, y_token_stride=128), 22, "very view"), (dict(y=0x20000 - 64), 22, "very view"), (dict(RES, y=0x50000), 22, "very view"),
    (dict(RES, residual_out=0x40000 + 16), 22, "very view"), (dict(RES, residual_f32=1, residual_out=0x10000), 22, "very view"),
])
def test_norm_refuses(kw, status, msg):
    st, err = norm(**kw)
    assert st == status and msg in err, (st, err)


@pytest.mark.parametrize("kw", [
    dict(), dict(y=0x10000), dict(RES), dict(RES, residual_out=0x40000), dict(RES, y=0x40000), dict(RES, residual_out=0x10000),
    dict(x_token_stride=0), dict(heads=2, y_head_stride=64, y_token_stride=128), dict(heads=2, y_head_stride=256, y_token_stride=64),
    dict(tokens=1, y_token_stride=0), dict(dim=32768, x_token_stride=1 << 31, y_token_stride=32768, y=1 << 44, tokens=2, weight=1 << 45),
])
def test_norm_accepts(kw):
    st, err = norm(**kw)
    assert st in DEVICE, (st, err)


def test_norm_of_no_rows_is_fine():
    assert norm(tokens=0, x=None, y=None, weight=None)[0] == 0


def route(logits=0x10000, dtype=2, stride=16, tokens=4, num=16, k=2, weights=0x20000, experts=0x30000):
    lib = capi.load()
    st = lib.w4a16_moe_route(logits, dtype, stride, tokens, num, k, 1, weights, experts, None)
    return st, capi.last_error(lib)


@pytest.mark.parametrize("kw,status,msg", [
    (dict(dtype=3), 20, "dtype"), (dict(num=0), 24, "num_experts"), (dict(num=1025), 24, "num_experts"), (dict(k=0), 24, "k must"),
    (dict(k=17), 24, "k must"), (dict(num=100, k=33), 24, "k must"), (dict(tokens=-1), 4, "int32"), (dict(tokens=1 << 60), 4, "int32"),
    (dict(stride=-1), 24, "row_stride"), (dict(logits=None), 1, "non-null"), (dict(logits=0x10002), 9, "aligned"),
    (dict(weights=0x10000), 22, "overlap"), (dict(experts=0x20004), 22, "overlap"),
])
def test_route_refuses(kw, status, msg):
    st, err = route(**kw)
    assert st == status and msg in err, (st, err)


def test_route_accepts():
    assert route()[0] in DEVICE and route(dtype=0, logits=0x10002)[0] in DEVICE and route(tokens=0, logits=None)[0] == 0


def test_order_of_gated_rows():
    gate, up = torch.arange(16.0)[:, None].expand(16, 3), 100 + torch.arange(16.0)[:, None].expand(16, 3)
    rows = interleave_gate_up(gate, up)[:, 0].tolist()
    assert rows == [*range(8), *range(100, 108), *range(8, 16), *range(108, 116)]
    assert torch.equal(interleave_gate_up(gate.t(), up.t(), dim=1), interleave_gate_up(gate, up).t())
    assert torch.equal(interleave_gate_up(gate.t(), up.t(), dim=-1), interleave_gate_up(gate, up).t())
    assert interleave_gate_up(gate[:, 0], up[:, 0]).tolist() == rows
    with pytest.raises(RuntimeError, match="multiple of 8"):
        interleave_gate_up(gate[:12], up[:12])
    with pytest.raises(RuntimeError, match="one shape"):
        interleave_gate_up(gate, up[:8])


def test_structures_are_laid_out_as_the_header_says(tmp_path):
    import os
    import subprocess
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    lines = []
    for c, struct in (("w4a16_epilogue", capi.Epilogue), ("w4a16_norm_args", capi.NormArgs), ("w4a16_moe_args", capi.MoeArgs)):
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        lines += [f'printf("%zu\\n", offsetof({c}, {name}));' for name, _ in struct._fields_]
    (tmp_path / "s.c").write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"w4a16.h\"\nint main(void) {\n" + "\n".join(lines) + "\nreturn 0; }\n")
    subprocess.run(["gcc", "-std=c99", "-pedantic", "-Wall", "-Werror", "-I", include, str(tmp_path / "s.c"), "-o", str(tmp_path / "s")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for struct in (capi.Epilogue, capi.NormArgs, capi.MoeArgs):
        want.append(ctypes.sizeof(struct))
        want += [getattr(struct, name).offset for name, _ in struct._fields_]
    assert got == want
