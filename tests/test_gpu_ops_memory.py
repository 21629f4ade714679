"""The operators where device memory runs out: torch's own error, on every path, and the
next call works."""
from __future__ import annotations

import pytest
import torch

from slideformer_amd import ops

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture
def no_memory(hip_device):
    """Leaves the allocator what it holds, and no more, until the test is over."""
    total = torch.cuda.get_device_properties(hip_device).total_memory

    def limit():
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        torch.cuda.set_per_process_memory_fraction(torch.cuda.memory_reserved(hip_device) / total, hip_device)
        held = []                                            # what is free between other tensors
        try:
            while True:
                held.append(torch.empty(1 << 24, dtype=torch.uint8, device=hip_device))
        except torch.OutOfMemoryError:
            return held

    yield limit
    torch.cuda.set_per_process_memory_fraction(1.0, hip_device)


@pytest.mark.parametrize("name", ["embedding", "embedding_grad", "rms_norm", "rms_norm_8bit", "rms_norm_grad",
                                  "linear_cross_entropy", "linear_cross_entropy_grad"])
@pytest.mark.parametrize("stream", [False, True])
def test_out_of_memory_is_torchs_error(hip_device, no_memory, name, stream):
    n, hidden = 16384, 2048
    side = torch.cuda.current_stream() if stream else None   # a stream that is named takes the path in Python
    weight = torch.zeros(8, hidden, dtype=BF16, device=hip_device)
    x = torch.zeros(n, hidden, dtype=BF16, device=hip_device)
    tokens = torch.zeros(n, dtype=torch.int64, device=hip_device)
    rstd = torch.ones(n, device=hip_device)
    call = {"embedding": lambda: ops.embedding(tokens, weight, stream=side),
            "embedding_grad": lambda: ops.embedding_grad(tokens, x, weight, stream=side),
            "rms_norm": lambda: ops.rms_norm(x, weight[0], stream=side),
            "rms_norm_8bit": lambda: ops.rms_norm_8bit(x, weight[0], stream=side),
            "rms_norm_grad": lambda: ops.rms_norm_grad(x, x, rstd, weight[0], stream=side),
            "linear_cross_entropy": lambda: ops.linear_cross_entropy(x, weight, tokens, stream=side),
            "linear_cross_entropy_grad": lambda: ops.linear_cross_entropy_grad(x, weight, tokens, stream=side)}[name]
    held = no_memory()                                       # less than 16 MiB is left in one place
    with pytest.raises(torch.OutOfMemoryError):
        call()
    del held
    torch.cuda.set_per_process_memory_fraction(1.0, hip_device)
    call()
    torch.cuda.synchronize()
