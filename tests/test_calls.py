"""The two editions of `Library.caller` (compiled, and in Python where the extension is not built) convert alike."""
import pytest
import torch


class Cuda:
    """Stands in for a CUDA tensor."""
    is_cuda = True

    def __init__(self, at=4096):
        self.at = at

    def data_ptr(self):
        return self.at


@pytest.fixture(params=["compiled", "python"])
def library(request, pkg):
    L = pkg.Library()
    if request.param == "python":
        L._compiled = None
    elif L._compiled is None:
        pytest.skip("the extension is not built")
    return L


def test_refusals_come_back_as_errors(library, pkg):
    f = library.caller("rms_norm_f16", Cuda)
    with pytest.raises(pkg.B200KError) as e:
        f(None, None, None, 128, 1 / 128, 1e-5, 4, None)
    assert e.value.code == -1 and "NULL" in e.value.message
    with pytest.raises(pkg.B200KError) as e:        # the float and the ints arrive in their places
        library.caller("kv_cache_append_hm_int4_f16", Cuda)(*[Cuda()] * 7, None, 8, 100, 64, 77, 1, 2, 800, 800, None)
    assert e.value.code == -2 and "head_dim 100" in e.value.message
    assert library.caller("kv_cache_append_hm_int4_f16", Cuda)(*[Cuda()] * 7, None, 8, 128, 64, 77, 0, 2, 1024, 1024, 7) == 0


def test_argument_kinds(library):
    f = library.caller("rms_norm_f16", Cuda)
    with pytest.raises(TypeError):
        f(None)
    with pytest.raises((TypeError, ValueError)):
        f(Cuda(), Cuda(), Cuda(), "x", 0.1, 0.1, 0, None)
    with pytest.raises(ValueError, match="argument weight must be a CUDA tensor"):
        f(Cuda(), torch.zeros(4), Cuda(), 4, 0.25, 1e-5, 0, None)
    # addresses as integers, a tensor-like of another type, a stream object, whole numbers of other types: no rows, no launch
    other = type("Other", (Cuda,), {})()
    stream = type("Stream", (), {"cuda_stream": 0})()
    for s in (None, 0, stream):
        assert f(4096, other, Cuda(), torch.tensor(4).item(), 0.25, 1, 0, s) == 0


def test_counts_and_sizes_are_not_statuses(library, pkg):
    size = library.caller("b200k_gemm_workspace_bytes", Cuda)(16, 4096, 4096)
    assert size == pkg.lib().call("b200k_gemm_workspace_bytes", 16, 4096, 4096) > 0
    assert library.caller("b200k_layer_launches_per_forward", Cuda)(None) == 0


def test_the_stream_may_be_left_out_or_named(library, pkg):
    seen = []

    def current():
        seen.append(1)
        return 0
    f = library.caller("rms_norm_f16", Cuda, current)
    args = (Cuda(), Cuda(), Cuda(), 4, 0.25, 1e-5, 0)
    assert f(*args) == 0 and len(seen) == 1
    assert f(*args, stream=None) == 0 and len(seen) == 2
    stream = type("Stream", (), {"cuda_stream": 0})()
    assert f(*args, stream=stream) == 0 and f(*args, 0) == 0 and f(*args, None) == 0 and len(seen) == 2
    assert f.__name__ == "rms_norm_f16" and "rms_norm_f16" in f.__doc__
    for bad, named in ((args[:-1], {}), ((*args, 0, 0), {}), (args, {"other": 0}), (args, {"stream": 0, "other": 0})):
        with pytest.raises(TypeError):
            f(*bad, **named)
    with pytest.raises(TypeError):                   # no stream provider, no name
        library.caller("rms_norm_f16", Cuda)(*args, stream=0)
    with pytest.raises(TypeError):
        library.caller("rms_norm_f16", Cuda)(*args)

    def broken():
        raise RuntimeError("no stream")
    with pytest.raises(RuntimeError, match="no stream"):
        library.caller("rms_norm_f16", Cuda, broken)(*args)
    assert library.caller("rms_norm_f16", Cuda, current) is f


def test_prelude_functions_are_callers(pkg):
    f = pkg.prelude.rms_norm_f32
    assert f is pkg.prelude.rms_norm_f32 and f.__name__ == "rms_norm_f32"
    with pytest.raises(TypeError):
        f(None)
    with pytest.raises(pkg.B200KError) as e:
        f(None, None, None, 4, 0.25, 1e-5, 1, 0)
    assert e.value.code == -1
