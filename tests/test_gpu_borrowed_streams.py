"""GPU: borrowed memory whose writer is still at work on the stream that it names: the library waits for that stream."""
import numpy as np
import pytest

import pytortto_amd as tt

pytestmark = pytest.mark.gpu
torch = pytest.importorskip('torch')


class _Named:
    def __init__(self, tensor, stream):
        self.tensor = tensor
        self.__cuda_array_interface__ = dict(tensor.__cuda_array_interface__, version=3, stream=stream)


@pytest.mark.parametrize('which', ['default', 'per thread', 'own'])
def test_the_operator_waits_for_the_writer(which):
    """Some 20 ms of copies on the writer's stream, and the values behind them."""
    z = np.random.default_rng(0).standard_normal((64, 1000)).astype(np.float32)
    want = (z - z.mean(1, keepdims=True)) / np.sqrt(z.var(1, keepdims=True) + 1e-5)
    values, wrong = torch.from_numpy(z).cuda(), torch.full((64, 1000), 5.0, device='cuda')
    large = torch.zeros(1 << 28, device='cuda')
    copy = torch.zeros(1 << 28, device='cuda')
    handle, stream = {'default': (1, torch.cuda.default_stream()), 'per thread': (2, torch.cuda.ExternalStream(2)),
                      'own': (None, torch.cuda.Stream())}[which]
    handle = handle or stream.cuda_stream
    tt.nn.functional.layer_norm(tt.as_tensor(_Named(values, None)), 1000).data.get()     # (everything is loaded by now)
    for _ in range(3):
        buffer = wrong.clone()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for _ in range(40):
                copy.copy_(large)
            buffer.copy_(values)
        got = tt.nn.functional.layer_norm(tt.as_tensor(_Named(buffer, handle)), 1000).data.get()
        np.testing.assert_allclose(got, want, atol=1e-5)
        assert stream.query()           # the writer is done by then
