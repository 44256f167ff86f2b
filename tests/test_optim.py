"""Host side of the AdamW over many tensors (mmearth_train_amd.optim): layout, code format, refusals, struct layouts. No GPU."""
import ctypes as C
import math
import os
import subprocess

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_moment_layout_starts_every_tensor_in_a_block_of_its_own():
    from mmearth_train_amd.optim import BLOCK, moment_layout
    offsets, size = moment_layout([1, 256, 0, 257, 5])
    assert offsets == [0, 256, 512, 512, 1024] and size == 1280 and BLOCK == 256


def test_codes_hold_what_the_format_says():
    from mmearth_train_amd.optim import quantize_moments
    gen = torch.Generator().manual_seed(1)
    m = torch.randn(64 * 256, generator=gen) * torch.exp(2 * torch.randn(64 * 256, generator=gen))
    v = m * m * torch.rand(64 * 256, generator=gen)
    v[300:310] = 0.0
    km, kv, sm, sv = quantize_moments(m, v)
    k, l = km.double().view(64, 256), kv.double().view(64, 256)
    mv, vv = k * k.abs() * (sm.double() / 127 ** 2)[:, None], l ** 4 * (sv.double() / 255 ** 4)[:, None]
    # half a code in the root: |sqrt(|m| / s) - k / 127| <= 0.5 / 127, |(v / s)^(1/4) - k / 255| <= 0.5 / 255 unless v was lifted to code 1
    a, b = (m.double().view(64, 256).abs() / sm.double()[:, None]).sqrt(), (v.double().view(64, 256) / sv.double()[:, None]) ** 0.25
    assert float((a - k.abs() / 127).abs().max()) <= 0.5 / 127 * (1 + 1e-12)
    assert float((b - l / 255)[l != 1].abs().max()) <= 0.5 / 255 * (1 + 1e-12)
    assert torch.equal(l == 0, v.view(64, 256) == 0) and torch.equal(torch.sign(k)[k != 0], torch.sign(m.double().view(64, 256))[k != 0])
    # the values have the same codes again, also from fp32
    again = quantize_moments(mv.float().reshape(-1), vv.float().reshape(-1))
    assert all(torch.equal(x, y) for x, y in zip((km, kv, sm, sv), again))


def test_codes_of_bad_and_empty_blocks():
    from mmearth_train_amd.optim import quantize_moments
    m, v = torch.zeros(1024), torch.zeros(1024)
    m[256], v[600] = float("inf"), float("nan")
    m[300] = 1.0
    km, kv, sm, sv = quantize_moments(m, v)
    assert not km.any() and not kv.any()
    assert [math.isnan(float(x)) for x in sm] == [False, True, False, False] and [math.isnan(float(x)) for x in sv] == [False, False, True, False]


@pytest.mark.parametrize("kw,what", [
    (dict(state_bits=16), "state_bits"), (dict(max_norm=0.0), "max_norm"), (dict(max_norm=float("inf")), "max_norm"), (dict(lr=-1.0), "lr"),
    (dict(lr=float("nan")), "lr"), (dict(lr=torch.tensor(1e-3)), "lr is a number"), (dict(eps=-1e-8), "eps"), (dict(weight_decay=-0.1), "weight_decay"),
    (dict(betas=(1.0, 0.9)), "betas"), (dict(betas=(0.9, -0.1)), "betas"),
])
def test_refused_settings(kw, what):
    from mmearth_train_amd.optim import AdamW
    with pytest.raises(ValueError, match=what):
        AdamW([torch.nn.Parameter(torch.zeros(4))], **kw)


def test_refused_parameters():
    from mmearth_train_amd.optim import AdamW
    mk = torch.nn.Parameter
    with pytest.raises(ValueError, match="GPU only"):
        AdamW([mk(torch.zeros(4))])
    with pytest.raises(ValueError, match="fp32, bf16 or fp16"):
        AdamW([mk(torch.zeros(4, dtype=torch.float64))])
    with pytest.raises(ValueError, match="densely"):
        AdamW([mk(torch.zeros(4, 4)[:, ::2])])
    with pytest.raises(ValueError, match="densely"):
        AdamW([mk(torch.zeros(1, 4).expand(4, 4).detach())])
    with pytest.raises(ValueError):
        AdamW([])


def test_dense_recognises_orders():
    from mmearth_train_amd.optim import _dense
    x = torch.zeros(3, 4, 5, 6)
    assert _dense(x) and _dense(x.permute(2, 0, 3, 1)) and _dense(x[:1]) and _dense(x.contiguous(memory_format=torch.channels_last)) and _dense(torch.zeros(()))
    assert not _dense(x[:, 1:]) and not _dense(x.expand(2, 3, 4, 5, 6)) and not _dense(x[..., ::2])


def test_library_refuses_bad_arguments(lib):
    """The C entry points return an error instead of launching: no GPU is touched."""
    from mmearth_train_amd import _lib
    one = (C.c_double * 5)(1e-3, 0.9, 0.99, 1e-8, 0.0)
    some = C.create_string_buffer(256)
    at = C.addressof(some)
    full = dict(tensors=at, chunks=at, chunk_first=at, steps=at, hyper=at, partials=at, norm_skip=at, m=at, v=at, ms=at, vs=at, max_norm=0.0, nt=1,
                npartials=1, bits=32)
    for bad in (dict(nt=0), dict(bits=16), dict(m=None), dict(bits=8, ms=None), dict(max_norm=1.0, partials=None), dict(tensors=None), dict(steps=None)):
        args = _lib.AdamwArgs(**{**full, **bad})
        assert lib.mpmae_adamw_multi(C.byref(args), at, one, 1, None) != 0, bad
    args = _lib.AdamwArgs(**full)
    assert lib.mpmae_adamw_multi(C.byref(args), None, one, 1, None) != 0
    assert lib.mpmae_adamw_multi(C.byref(args), at, one, 0, None) != 0
    assert lib.mpmae_adamw_values(at, at, at, at, at, at, 255, None) != 0
    assert lib.mpmae_adamw_values(at, at, at, at, at, at, -256, None) != 0
    assert lib.mpmae_adamw_values(at, at, at, at, at, at, 0, None) == 0


def test_structs_match_the_header(tmp_path):
    from mmearth_train_amd import _lib, optim
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "mpmae_hip.h"\nint main(void) { printf("%zu %zu %d %d %zu %zu\\n", sizeof(MpmaeAdamwArgs), sizeof(MpmaeAdamwTensor),'
                   " MPMAE_ADAMW_HYPER_BYTES, MPMAE_ADAMW_NORM_BLOCKS, offsetof(MpmaeAdamwArgs, max_norm), offsetof(MpmaeAdamwTensor, group)); return 0; }\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(_lib.AdamwArgs), optim._TABLE.itemsize, _lib.ADAMW_HYPER_BYTES, _lib.ADAMW_NORM_BLOCKS, _lib.AdamwArgs.max_norm.offset,
                   optim._TABLE.fields["group"][1]]


def test_native_reader_refuses_what_it_cannot_address():
    """csrc/host_tensors.cpp raises instead of handing an address on: everything here is on the CPU, so nothing gets as far as an address."""
    from mmearth_train_amd import _lib, optim
    host = _lib.host_tensors()
    table, out = np.zeros(1, optim._TABLE), np.zeros(2, np.uint64)
    with pytest.raises(ValueError, match="device"):
        host.gather([torch.nn.Parameter(torch.zeros(3))], table.ctypes.data, 0, out.ctypes.data, out.ctypes.data, True)
    with pytest.raises(ValueError, match="not a tensor"):
        host.gather([3], table.ctypes.data, 0, out.ctypes.data, out.ctypes.data, True)
    assert host.gather([], table.ctypes.data, 0, out.ctypes.data, out.ctypes.data, True) == (0, False, None)


def _reader_state(params):
    from mmearth_train_amd import optim
    table = np.zeros(len(params), optim._TABLE)
    table["n"], table["p"] = [p.numel() for p in params], [p.data_ptr() for p in params]
    return table, np.zeros(len(params), np.uint64), np.zeros(len(params), np.uint64)


@pytest.mark.parametrize("count,refused", [(2, 1), (2, 0), (1, 0), (3, 2)])
def test_a_refused_list_does_not_lose_what_has_moved(count, refused):
    """The native reader over host memory (device -1): parameters move, one gradient is refused, it is put right: the next call still reports the move, and the
    refusal itself left addresses, orders and versions alone."""
    from mmearth_train_amd import _lib
    host = _lib.host_tensors()
    params = [torch.nn.Parameter(torch.ones(300 + i)) for i in range(count)]
    for p in params:
        p.grad = torch.ones_like(p)
    table, out, orders = _reader_state(params)
    read = lambda: host.gather(params, table.ctypes.data, -1, out.ctypes.data, orders.ctypes.data, True)  # noqa: E731
    assert read() == (count, False, None)
    old = [p.data for p in params]                            # (alive: no new tensor can take their place)
    for p in params:
        p.data = p.data.clone()
    good = params[refused].grad
    for bad in (torch.ones_like(good).to_sparse(), None):
        if bad is None:                                       # of another shape, given behind autograd's back
            params[refused].grad = good
            params[refused].grad.data = torch.ones(7)
        else:
            params[refused].grad = bad
        keep, versions = (table.copy(), orders.copy()), [p._version for p in params]
        with pytest.raises(ValueError, match=f"parameter {refused} has a"):
            read()
        assert np.array_equal(table, keep[0]) and np.array_equal(orders, keep[1]) and versions == [p._version for p in params]
    params[refused].grad = torch.ones_like(params[refused])
    assert read() == (count, True, None)
    assert table["p"].tolist() == [p.data_ptr() for p in params] and out.tolist() == [p.grad.data_ptr() for p in params]
    assert not set(table["p"].tolist()) & {p.data_ptr() for p in old}
    assert read() == (count, False, None)


def test_lists_are_compared_object_for_object():
    from mmearth_train_amd import _lib
    same = _lib.host_tensors().same_lists
    a, b, c = (torch.nn.Parameter(torch.zeros(3)) for _ in range(3))
    group = lambda *ps: {"params": list(ps), "lr": 1.0}  # noqa: E731
    assert same([group(a, b), group(c)], [a, b, c], [2, 1]) and same([], [], []) and same([group(), group(a)], [a], [0, 1])
    for groups in ([group(a, b), group(b)], [group(b, a), group(c)], [group(a, c), group(b)], [group(a), group(b, c)], [group(c), group(a, b)], [group(a, b)],
                   [group(a, b), group(c), group()], [group(a, b), group()], [group(a, b), {"params": (c,)}], [group(a, b), 3]):
        assert not same(groups, [a, b, c], [2, 1])
    assert not same([group(a)], [a, b], [1]) and not same([group(a, b)], [a], [2])
    with pytest.raises(TypeError):
        same([], [], 3)


def test_a_parameter_of_inference_mode_is_refused_before_anything_is_written():
    """It has no version counter, and the error that counting it raises would come half way through the list."""
    from mmearth_train_amd import _lib
    host = _lib.host_tensors()
    with torch.inference_mode():
        second = torch.nn.Parameter(torch.ones(7))
        second.grad = torch.ones(7)
    params = [torch.nn.Parameter(torch.ones(300)), second]
    params[0].grad = torch.ones(300)
    table, out, orders = _reader_state(params)
    keep = table.copy()
    params[0].data = params[0].data.clone()
    with pytest.raises(ValueError, match="parameter 1 was made in inference mode"):
        host.gather(params, table.ctypes.data, -1, out.ctypes.data, orders.ctypes.data, True)
    assert np.array_equal(table, keep) and not orders.any() and params[0]._version == 0


def test_a_negated_gradient_is_copied_not_addressed():
    """The imaginary part of a conjugate: its memory holds the values with the other sign."""
    from mmearth_train_amd import _lib
    host = _lib.host_tensors()
    p = torch.nn.Parameter(torch.ones(1))
    p.grad = torch.tensor([1 + 2j]).conj().imag
    assert p.grad.is_neg() and float(p.grad) == -2.0
    table, out, orders = _reader_state([p])
    assert host.gather([p], table.ctypes.data, -1, out.ctypes.data, orders.ctypes.data, True) == (1, False, [0]) and out[0] == 0
    q = torch.nn.Parameter(torch.tensor([1 + 2j]).conj().imag.detach())
    if q.is_neg():
        with pytest.raises(ValueError, match="dense"):
            host.gather([q], table.ctypes.data, -1, out.ctypes.data, np.zeros(1, np.uint64).ctypes.data, True)


def test_library_refuses_settings_that_no_update_has(lib):
    """hipErrorInvalidValue is 1; what is let through fails here for want of a GPU, with another error."""
    from mmearth_train_amd import _lib
    some = C.create_string_buffer(256)
    at = C.addressof(some)
    args = _lib.AdamwArgs(tensors=at, chunks=at, chunk_first=at, steps=at, hyper=at, partials=at, norm_skip=at, m=at, v=at, ms=at, vs=at, max_norm=0.0, nt=1, npartials=1, bits=32)
    nan, inf = float("nan"), float("inf")
    for bad in ((-1e-3, 0.9, 0.99, 1e-8, 0.0), (nan, 0.9, 0.99, 1e-8, 0.0), (inf, 0.9, 0.99, 1e-8, 0.0), (1e-3, 1.0, 0.99, 1e-8, 0.0), (1e-3, 0.9, 1.0, 1e-8, 0.0),
                (1e-3, -0.1, 0.99, 1e-8, 0.0), (1e-3, 0.9, nan, 1e-8, 0.0), (1e-3, 0.9, 0.99, -1e-8, 0.0), (1e-3, 0.9, 0.99, 1e-8, inf)):
        groups = (C.c_double * 10)(1e-3, 0.9, 0.99, 1e-8, 0.0, *bad)
        assert lib.mpmae_adamw_multi(C.byref(args), at, groups, 2, None) == 1, bad


@pytest.fixture(scope="module")
def lib():
    from mmearth_train_amd import _lib
    if not os.path.isfile(_lib.LIB_PATH):
        import __graft_entry__ as g
        g.build()
    return _lib.load()
