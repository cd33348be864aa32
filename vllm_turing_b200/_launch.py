"""Launches a C entry on the device its tensors live on, on that device's current stream."""
import torch


def launch(name, fn, device, *args):
    """fn(*args, stream) with `device` current; raises on a non-zero status."""
    i = device.index
    if i == torch.cuda.current_device():
        rc = fn(*args, torch.cuda.current_stream().cuda_stream)
    else:
        with torch.cuda.device(i):
            rc = fn(*args, torch.cuda.current_stream().cuda_stream)
    if rc != 0:
        raise RuntimeError(f"{name} failed: {rc}")


def need(ok, what):
    if not ok:
        raise ValueError(what)


def same_device(what, *tensors):
    """Every given tensor is a CUDA tensor of the first one's device."""
    d = tensors[0].device
    if d.type != "cuda" or any(t is not None and t.device != d for t in tensors):
        raise ValueError(f"{what}: CUDA tensors of one device are needed, got "
                         f"{[str(t.device) for t in tensors if t is not None]}")
    return d


def dtype_code(what, t, *others):
    """0 fp16 / 1 bf16, the same for every given tensor."""
    if t.dtype not in (torch.float16, torch.bfloat16) or any(o is not None and o.dtype != t.dtype for o in others):
        raise TypeError(f"{what}: one dtype, float16 or bfloat16, got "
                        f"{[str(x.dtype) for x in (t, *others) if x is not None]}")
    return 0 if t.dtype == torch.float16 else 1


def vector(t, dtype, n):
    """A contiguous 1-D tensor of n elements."""
    return t.dtype == dtype and t.dim() == 1 and t.shape[0] == n and t.is_contiguous()
