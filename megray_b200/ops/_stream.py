"""The current CUDA stream as the handle the native library takes."""
import torch


def raw_stream(index: int = None) -> int:
    """``torch.cuda.current_stream().cuda_stream`` without building a Stream object; ``index`` is the current
    device where the caller knows it."""
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if index is None else index)
