"""GPU: blocks of arrays that torch works on."""
import ctypes

import numpy as np
import pytest

import pytortto_amd as tt
from pytortto_amd import _hip
from pytortto_amd.xparray import hiparray

pytestmark = pytest.mark.gpu
torch = pytest.importorskip('torch')


def _pooled():
    used, pooled, workspace = ctypes.c_size_t(), ctypes.c_size_t(), ctypes.c_size_t()
    _hip.call('tt_mem_stats', ctypes.byref(used), ctypes.byref(pooled), ctypes.byref(workspace))
    return pooled.value


def _theirs(array):
    return torch.as_tensor(array, device='cuda')


def _export_and_drop(times, n=4):
    for _ in range(times):
        _theirs(hiparray.empty((n,)))


def test_a_block_is_not_reused_before_torch_has_read_it():
    n = (1 << 20) + 12345               # (a size that nothing else here has)
    values = np.random.default_rng(0).standard_normal(n).astype(np.float32)
    work = torch.randn(8192, 8192, device='cuda').bfloat16()
    out = work @ work
    array = hiparray(values)
    at, view = array.ptr, _theirs(array)
    torch.cuda.synchronize()
    for _ in range(40):                 # some 40 ms on the default stream, and the copy behind them
        torch.mm(work, work, out=out)
    kept = view.clone()
    del array, view
    _export_and_drop(70)                # enough of them that blocks are taken back
    taken = [hiparray.empty((n,)) for _ in range(3)]
    assert at in [a.ptr for a in taken]
    for a in taken:
        a.fill(7.0)
    tt.cuda.synchronize()
    np.testing.assert_array_equal(kept.cpu().numpy(), values)


def test_results_that_torch_drops_at_once():
    """A loop as a program runs it: results are read by torch behind other work of its own, and dropped."""
    rng = np.random.default_rng(1)
    z = [rng.standard_normal((64, 4096)).astype(np.float32) for _ in range(4)]
    x = [tt.Tensor(hiparray(a)) for a in z]
    want = [(a - a.mean(1, keepdims=True)) / np.sqrt(a.var(1, keepdims=True) + 1e-5) for a in z]
    work = torch.randn(4096, 4096, device='cuda').bfloat16()
    out = work @ work
    sums = [torch.zeros((64, 4096), device='cuda') for _ in z]
    for _ in range(50):
        for i, t in enumerate(x):
            y = tt.nn.functional.layer_norm(t, 4096)
            tt.cuda.synchronize()
            torch.mm(work, work, out=out)
            sums[i] += _theirs(y.data)
            del y
    torch.cuda.synchronize()
    for s, v in zip(sums, want):
        np.testing.assert_allclose(s.cpu().numpy(), 50 * v, atol=50 * 2e-5)


def test_the_pool_does_not_grow():
    _export_and_drop(300, 50000)
    before = _pooled()
    _export_and_drop(1000, 50000)
    assert _pooled() <= before + 65 * 50176 * 4
    _hip.call('tt_empty_cache')
    assert _pooled() == 0


def test_twice_is_refused():
    p = ctypes.c_void_p()
    _hip.call('tt_malloc', ctypes.byref(p), 100)
    _hip.call('tt_free_exported', p)
    with pytest.raises(RuntimeError, match='tt_free_exported: .* freed twice'):
        _hip.call('tt_free_exported', p)
    _hip.call('tt_free_exported', None)


def test_the_stream_that_the_interface_names():
    """Work on the default stream that waits for the named one finds the result, without any other wait."""
    z = np.random.default_rng(2).standard_normal((4096, 4096)).astype(np.float32)
    x = tt.Tensor(hiparray(z))
    theirs = torch.empty((4096, 4096), device='cuda')
    torch.cuda.synchronize()
    tt.cuda.synchronize()
    for _ in range(3):
        y = x
        for _ in range(20):
            y = tt.nn.functional.layer_norm(y, 4096)
        handle = y.data.__cuda_array_interface__['stream']
        assert handle == _hip.stream() and handle > 2
        torch.cuda.default_stream().wait_stream(torch.cuda.ExternalStream(handle))
        theirs.copy_(_theirs(y.data))
        want = y.data.get()
        np.testing.assert_array_equal(theirs.cpu().numpy(), want)
        theirs.zero_()
