"""Results given with out=: autograd learns that they were written."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16 = torch.float16


def calls():
    import tensorcoreptx_b200 as t
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(40, 64, generator=g, device=DEV).to(F16)
    W = torch.randn(2, 24, 64, generator=g, device=DEV).to(F16)
    o = torch.tensor([0, 13, 40], dtype=torch.int32, device=DEV)
    q, s = t.quantize_rows_int8(x)
    B, sb = t.quantize_rows_int8(W)
    return {
        "gemm_grouped": lambda out: t.gemm_grouped(x, W, o, out=out),
        "gemm_int8_grouped": lambda out: t.gemm_int8_grouped(q, B, o, s, sb, out=out),
        "linear_int8_grouped": lambda out: t.linear_int8_grouped(x, B, o, sb, out=out),
    }


NAMES = ["gemm_grouped", "gemm_int8_grouped", "linear_int8_grouped"]


@pytest.mark.parametrize("name", NAMES)
def test_a_buffer_that_a_backward_pass_needs_is_seen_to_change(name):
    call = calls()[name]
    buf = torch.randn(40, 24, device=DEV).to(F16)
    w = torch.randn(40, 24, device=DEV).to(F16).requires_grad_(True)
    y = (w * buf).sum()  # keeps buf
    version = buf._version
    assert call(buf) is buf and buf._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()


@pytest.mark.parametrize("name", NAMES)
def test_a_slice_of_a_buffer_counts_as_the_buffer(name):
    call = calls()[name]
    buf = torch.zeros(3, 40, 24, device=DEV, dtype=F16)
    version = buf._version
    got = call(buf[1])
    assert buf._version > version and torch.equal(got, call(None)) and torch.equal(buf[1], got)
    assert (buf[0] == 0).all() and (buf[2] == 0).all()


@pytest.mark.parametrize("name", NAMES)
def test_a_result_that_requires_grad_is_refused(name):
    call = calls()[name]
    buf = torch.full((40, 24), 7.0, device=DEV, dtype=F16).requires_grad_(True)
    for out in (buf, buf * 1):
        with pytest.raises(RuntimeError, match="out must not require grad"):
            call(out)
        assert (out == 7).all()
    with torch.no_grad():  # as torch's own out= forms: written, and counted
        version = buf._version
        assert torch.equal(call(buf), call(None)) and buf._version > version


@pytest.mark.parametrize("name", NAMES)
def test_inference_tensors(name):
    call = calls()[name]
    with torch.inference_mode():
        buf = torch.zeros(40, 24, device=DEV, dtype=F16)
        assert torch.equal(call(buf), call(None))
        buf.zero_()
    with pytest.raises(RuntimeError, match="nference"):
        call(buf)
    assert (buf == 0).all()
