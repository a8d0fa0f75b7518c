"""inf_check_status beside a capture."""
import pytest

import infb200 as I

pytestmark = pytest.mark.gpu


def test_refused_on_a_capturing_stream(cuda):
    """The call is refused, the capture goes on, and the status word keeps what it held."""
    torch = cuda
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    x = torch.zeros(8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    code = 0
    with torch.cuda.graph(graph):
        x += 1
        try:
            I.check_status(status.data_ptr(), torch.cuda.current_stream().cuda_stream)
        except I.InfError as e:
            code = e.code
        x += 2
    assert code == 4
    status.fill_(3)
    graph.replay()
    torch.cuda.synchronize()
    assert x.tolist() == [3.0] * 8 and int(status) == 3
    with pytest.raises(I.InfError) as e:
        I.check_status(status.data_ptr())
    assert e.value.code == 11 and int(status) == 0
