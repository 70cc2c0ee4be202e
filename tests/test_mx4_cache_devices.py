"""Every operand of the block-scaled operators has to be on the current device: a pointer of another GPU's memory must not
reach a kernel.  On the host, with stand-ins for tensors of two devices; nothing is launched."""
import pytest
import torch

from fufft_b200 import ops


class Here(torch.Tensor):
    """passes for a tensor on cuda:0"""
    is_cuda = True

    def get_device(self):
        return 0


class There(torch.Tensor):
    """passes for a tensor on cuda:1"""
    is_cuda = True

    def get_device(self):
        return 1


class Launched(Exception):
    pass


class Library:
    """stands in for the shared library: answers sizes, and says when a call would have launched"""

    def fufft_cache_conv_workspace(self, *_):
        return 64

    def __getattr__(self, name):
        def call(*_):
            raise Launched(name)
        return call


@pytest.fixture(autouse=True)
def on_device_0(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 0, raising=False)
    monkeypatch.setattr(ops, "lib", Library)


def _tensors(where):
    """operands by name, each of the class that `where` gives it"""
    f32, i32, u8 = (lambda *s: torch.zeros(*s)), (lambda *s: torch.zeros(*s, dtype=torch.int32)), (lambda *s: torch.zeros(*s, dtype=torch.uint8))
    t = {"x": f32(8, 64), "x4": f32(4, 64), "bias": f32(16), "y": f32(8, 16), "codes": u8(16, 128), "scales": u8(1, 2, 32, 4, 4),
         "a_codes": u8(8, 128), "a_scales": u8(1, 2, 32, 4, 4),
         "wide": f32(8, 64), "cache_codes": u8(4, 16, 64), "cache_scales": u8(4, 16, 2), "table": i32(2, 2), "cu": i32(3), "starts": i32(2),
         "lengths": i32(2), "taps": f32(8, 64), "gate": f32(2, 64), "out": f32(2, 64), "workspace": u8(64)}
    return {k: v.as_subclass(where(k)) for k, v in t.items()}


def _calls(t):
    """name -> (call, its operands)"""
    w = lambda: ops.Mx4(t["codes"], t["scales"], 16, 64)                # noqa: E731
    a = lambda: ops.Mx4(t["a_codes"], t["a_scales"], 8, 64)             # noqa: E731
    cache = lambda: ops.SeqCache(t["cache_codes"], t["cache_scales"], t["table"], "mx8")  # noqa: E731
    kept = ("cache_codes", "cache_scales", "table")
    return {
        "quantize": (lambda: ops.mx4_quantize(t["x"]), ("x",)),
        "quantize_both": (lambda: ops.mx4_quantize_both(t["x"]), ("x",)),
        "dequantize": (lambda: ops.mx4_dequantize(a(), out=t["wide"]), ("a_codes", "a_scales", "wide")),
        "matmul": (lambda: ops.mx4_matmul(a(), w(), torch.float32, t["bias"], out=t["y"]),
                   ("a_codes", "a_scales", "codes", "scales", "bias", "y")),
        "linear": (lambda: ops.mx4_linear(t["x"], w(), t["bias"]), ("x", "codes", "scales", "bias")),
        "linear of few rows": (lambda: ops.mx4_linear(t["x4"], w(), t["bias"]), ("x4", "codes", "scales", "bias")),
        "append": (lambda: ops.cache_append(cache(), t["x"], t["cu"], t["starts"]), (*kept, "x", "cu", "starts")),
        "read": (lambda: ops.cache_read(cache(), t["cu"], t["starts"], 8, torch.float32, out=t["wide"]), (*kept, "cu", "starts", "wide")),
        "read_channels": (lambda: ops.cache_read_channels(cache(), t["starts"], t["lengths"], 16), (*kept, "starts", "lengths")),
        "conv": (lambda: ops.cache_conv(cache(), t["lengths"], t["taps"], t["gate"], torch.float32, t["out"], t["workspace"]),
                 (*kept, "lengths", "taps", "gate", "out", "workspace")),
    }


NAMES = list(_calls(_tensors(lambda k: Here)))


@pytest.mark.parametrize("name", NAMES)
def test_operands_on_the_current_device_launch(name):
    call, _ = _calls(_tensors(lambda k: Here))[name]
    with pytest.raises(Launched):
        call()


@pytest.mark.parametrize("name", NAMES)
def test_an_operand_elsewhere_is_refused(name):
    for operand in _calls(_tensors(lambda k: Here))[name][1]:
        call, _ = _calls(_tensors(lambda k: There if k == operand else Here))[name]
        with pytest.raises(ValueError, match="cuda:1"):
            call()


@pytest.mark.parametrize("name", NAMES)
def test_all_operands_elsewhere_are_refused(name):
    call, _ = _calls(_tensors(lambda k: There))[name]
    with pytest.raises(ValueError, match="current device is cuda:0"):
        call()


@pytest.mark.parametrize("elsewhere", ["a", "b", "both"])
def test_a_matrix_elsewhere_is_refused(elsewhere):
    """whole matrices of another device, which their constructor has no reason to refuse"""
    here, there = _tensors(lambda k: Here), _tensors(lambda k: There)
    t = there if elsewhere in ("a", "both") else here
    a = ops.Mx4(t["a_codes"], t["a_scales"], 8, 64)
    t = there if elsewhere in ("b", "both") else here
    b = ops.Mx4(t["codes"], t["scales"], 16, 64)
    for out in (None, here["y"], there["y"]):
        with pytest.raises(ValueError, match="cuda:1"):
            ops.mx4_matmul(a, b, torch.float32, out=out)
    if elsewhere != "a":
        for x in (here["x"], here["x4"], there["x"], there["x4"]):
            with pytest.raises(ValueError, match="cuda:1"):
                ops.mx4_linear(x, b)
    if elsewhere != "b":
        for out in (None, here["wide"], there["wide"]):
            with pytest.raises(ValueError, match="cuda:1"):
                ops.mx4_dequantize(a, out=out)


@pytest.mark.parametrize("name", ["append", "read", "read_channels", "conv"])
def test_a_cache_elsewhere_is_refused(name):
    t = {k: (There if k in ("cache_codes", "cache_scales", "table") else Here) for k in _tensors(lambda k: Here)}
    call, _ = _calls(_tensors(t.get))[name]
    with pytest.raises(ValueError, match="cuda:1"):
        call()


def test_tensors_of_the_host_are_refused():
    t = _tensors(lambda k: torch.Tensor)
    for call, operands in _calls(t).values():
        with pytest.raises(ValueError):
            call()
    for name, (_, operands) in _calls(_tensors(lambda k: Here)).items():
        for operand in operands:
            call, _ = _calls(_tensors(lambda k: torch.Tensor if k == operand else Here))[name]
            with pytest.raises(ValueError):
                call()
