"""Host side of the int8 linear layer: refusals, struct layout. No GPU."""
import ctypes as C
import os
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("w,b,what", [
    (torch.zeros(4), None, "matrix"), (torch.zeros(0, 4), None, "matrix"), (torch.zeros(4, 0), None, "matrix"),
    (torch.zeros(4, 4, dtype=torch.float64), None, "fp32, bf16 or fp16"), (torch.zeros(4, 4, dtype=torch.int8), None, "fp32, bf16 or fp16"),
    (torch.zeros(1, 131072), None, "at most 131071"), (torch.zeros(4, 4), torch.zeros(5), "bias"), (torch.zeros(4, 4), None, "GPU only"),
])
def test_refused_weights(w, b, what):
    from mmearth_train_amd.int8 import quantize_weight
    with pytest.raises(ValueError, match=what):
        quantize_weight(w, b)


def test_library_refuses_bad_arguments():
    """An error instead of a launch: no GPU is touched."""
    from mmearth_train_amd import _lib
    lib = _lib.load()
    room = C.create_string_buffer(4096)
    at = (C.addressof(room) + 15) & ~15
    for bad in ((3, at, 8, 1, 8, at, 128, at), (0, None, 8, 1, 8, at, 128, at), (0, at, 8, 0, 8, at, 128, at), (0, at, 8, 1, 0, at, 128, at), (0, at, -1, 1, 8, at, 128, at),
                (0, at, 8, 1, 8, at, 64, at), (0, at, 8, 1, 129, at, 128, at), (0, at, 8, 1, 8, at + 4, 128, at), (0, at, 8, 1, 131072, at, 131072, at)):
        assert lib.mpmae_quant_i8(*bad, None) != 0, bad
    full = dict(x=at, q=at, sx=at, w=at, sw=at, bias=None, y=at, ldx=8, ldy=4, M=1, N=4, K=8, ldq=128, ldw=128)
    for bad in (dict(N=0), dict(w=None), dict(sw=None), dict(y=None), dict(ldy=3), dict(ldw=256), dict(w=at + 8), dict(M=-1), dict(ldq=100)):
        assert lib.mpmae_linear_i8(0, C.byref(_lib.I8Args(**{**full, **bad})), None) != 0, bad
    assert lib.mpmae_linear_i8(5, C.byref(_lib.I8Args(**full)), None) != 0
    assert lib.mpmae_linear_i8(0, None, None) != 0


def test_rows_of_codes_are_k_rounded_up_and_no_longer():
    """Wider rows would split k in more parts than the workspace was sized for (64 x 3900 -> 1000: none by K, four by rows of 4096 bytes) and leave the padding of
    rows of fewer than eight elements unwritten. hipErrorInvalidValue is 1; a call that is let through fails here for want of a GPU, with another error."""
    from mmearth_train_amd import _lib
    lib = _lib.load()
    room = C.create_string_buffer(4096)
    at = (C.addressof(room) + 15) & ~15
    assert lib.mpmae_linear_i8_part_bytes(64, 1000, 3900) == 0 and lib.mpmae_linear_i8_part_bytes(64, 1000, 4096) == 4 * 4 * 64 * 1000
    for k, wide in ((3900, 4096), (3900, 3968 + 128), (1, 256), (7, 256), (128, 256), (129, 384), (100, 0), (100, -128)):
        assert lib.mpmae_quant_i8(0, at, k, 1, k, at, wide, at, None) == 1, (k, wide)
        args = _lib.I8Args(x=at, q=at, sx=at, w=at, sw=at, bias=None, y=at, part=at, ldx=k, ldy=1000, M=64, N=1000, K=k, ldq=wide, ldw=wide)
        assert lib.mpmae_linear_i8(0, C.byref(args), None) == 1, (k, wide)
    # (products whose workspace is missing are refused, whatever their size)
    args = _lib.I8Args(x=at, q=at, sx=at, w=at, sw=at, bias=None, y=at, part=None, ldx=4096, ldy=1000, M=64, N=1000, K=4096, ldq=4096, ldw=4096)
    assert lib.mpmae_linear_i8(0, C.byref(args), None) == 1


def test_struct_matches_the_header(tmp_path):
    from mmearth_train_amd import _lib
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "mpmae_hip.h"\nint main(void) { printf("%zu %zu %zu\\n", sizeof(MpmaeI8Args), offsetof(MpmaeI8Args, ldx), '
                   "offsetof(MpmaeI8Args, ldw)); return 0; }\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(_lib.I8Args), _lib.I8Args.ldx.offset, _lib.I8Args.ldw.offset]


def test_module_tree_and_moves():
    from mmearth_train_amd.int8 import Int8Linear
    m = Int8Linear(100, 7)
    assert set(m.state_dict()) == {"q", "scale", "bias"} and m.q.shape == (7, 128)
    assert set(Int8Linear(100, 7, bias=False).state_dict()) == {"q", "scale"}
    h = m.half()
    assert h.scale.dtype == torch.float32 and h.bias.dtype == torch.float32 and h.q.dtype == torch.int8
    assert m.to("meta").q.device.type == "meta"


def test_rows_of_any_input():
    from mmearth_train_amd.int8 import _rows
    x = torch.arange(240.0).reshape(4, 6, 10)
    for v, ld in ((x, 10), (x[0], 10), (x[0, :, :7], 10), (x[0, 0], 10), (x[:, 0], 60)):
        r, m, d = _rows(v, v.shape[-1])
        assert r.shape == (m, v.shape[-1]) and (d == ld or m == 1) and (v.shape[-1] == 1 or r.stride(1) == 1)
        assert torch.equal(r, v.reshape(-1, v.shape[-1]))
    r, m, d = _rows(x[0].t(), 6)
    assert r.stride(1) == 1 and torch.equal(r, x[0].t())


def test_a_cpu_input_is_refused_and_modules_copy():
    import copy
    import pickle
    from mmearth_train_amd.int8 import Int8Linear
    m = Int8Linear(100, 7)
    with pytest.raises(ValueError, match="is on cpu"):
        m(torch.zeros(2, 100))
    for other in (copy.deepcopy(m), pickle.loads(pickle.dumps(m))):
        assert other.q.data_ptr() != m.q.data_ptr() and (other._weight is None or other._weight.q is other.q)


def test_the_call_is_an_operator_that_tracing_sees():
    """On tensors without memory: shapes come out of the operator's own rule, and a graph holds the operator instead of the empty tensor that it fills."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    from mmearth_train_amd.int8 import Int8Linear, Int8Weight, linear_int8, load_ops
    load_ops()
    m = Int8Linear(100, 7, device="meta")
    with torch.no_grad():
        y = m(torch.zeros(2, 3, 100, device="meta", dtype=torch.float16))
    assert y.shape == (2, 3, 7) and y.dtype == torch.float16 and y.is_meta
    with pytest.raises(ValueError, match="end in 100"):
        m(torch.zeros(2, 99, device="meta"))
    q, scale = torch.ops.mpmae.quantize_int8(torch.zeros(7, 100, device="meta"))
    assert q.shape == (7, 128) and q.dtype == torch.int8 and scale.shape == (7,) and scale.dtype == torch.float32
    with FakeTensorMode():
        for device in ("meta", "cuda"):
            new = lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device=device)  # noqa: E731, B023
            w = Int8Weight(new(7, 128, dtype=torch.int8), new(7), new(7), 100)
            graph = make_fx(lambda x: linear_int8(x, w) * 2)(new(5, 100)).graph  # noqa: B023
            called = [n.target for n in graph.nodes if n.op == "call_function"]
            assert torch.ops.mpmae.linear_int8.default in called and not any("empty" in str(t) for t in called), called


def test_derivatives_are_refused_not_dropped():
    import torch.autograd.forward_ad as fwad
    from mmearth_train_amd.int8 import Int8Linear
    m, x = Int8Linear(100, 7), torch.ones(2, 100)
    with pytest.raises(RuntimeError, match="no backward"):
        m(x.clone().requires_grad_())
    with fwad.dual_level():
        with pytest.raises(RuntimeError, match="no derivative"):
            m(fwad.make_dual(x, torch.ones_like(x)))
    with pytest.raises(RuntimeError, match="no derivative"):
        torch.func.jvp(m, (x,), (x,))
    with pytest.raises(RuntimeError, match="no backward"):
        torch.func.grad(lambda x: m(x).sum())(x)
    with pytest.raises(ValueError, match="is on cpu"):          # (without either, the device is what is wrong here)
        m(x)
