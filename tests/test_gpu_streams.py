"""Operators on tensors that torch writes and reads on its own stream: the library's stream waits for it and
it waits for the library's."""
import numpy as np
import pytest

import eshkol_b200 as eb
from eshkol_b200 import api
from test_gpu_norm_logprobs import done, kinds

pytestmark = pytest.mark.gpu


def test_torchs_stream_before_and_after(gpu_lib):
    import torch
    t, tag, wt, u, half = kinds("f32")
    rows, n = 400, 600
    x, y = torch.zeros(rows, n, device="cuda"), torch.zeros(rows, n, device="cuda")
    w = torch.eye(n, device="cuda") * 2.0
    torch.cuda.synchronize()
    library, side = torch.cuda.ExternalStream(api.stream_handle()), torch.cuda.Stream()
    got = []
    with torch.cuda.stream(side):
        for turn in range(5):
            torch.cuda._sleep(20_000_000)  # some ten milliseconds before the inputs are written
            x.fill_(float(turn + 1))
            library.wait_stream(torch.cuda.current_stream())
            eb.linear_device(x.data_ptr(), w.data_ptr(), y.data_ptr(), rows, n, n, eb.make_linear_opts(tag))
            torch.cuda.current_stream().wait_stream(library)
            got.append(y.clone())
            y.fill_(float("nan"))
    torch.cuda.synchronize()
    done()
    for turn, v in enumerate(got):
        assert np.array_equal(v.cpu().numpy(), np.full((rows, n), 2.0 * (turn + 1), dtype=np.float32))
