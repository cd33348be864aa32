"""Launches a C entry on the device its tensors live on, on that device's current stream, and the refusals the entries
share. The calls below run once per layer of a decode step, so what every call does is kept to a few plain comparisons;
a refused call explains itself on its own path."""
import torch

# the current device and stream without building Python objects for them (2 x 3 us a call otherwise)
_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_stream = (getattr(torch._C, "_cuda_getCurrentRawStream", None)
           or (lambda i: torch.cuda.current_stream(i).cuda_stream))


def launch(name, fn, index, *args):
    """fn(*args, stream) with device `index` current; raises on a non-zero status."""
    if index == _device():
        rc = fn(*args, _stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _stream(index))
    if rc != 0:
        raise RuntimeError(f"{name} failed: {rc}")


def need(ok, what):
    if not ok:
        raise ValueError(what)


def refuse_devices(what, *tensors):
    raise ValueError(f"{what}: CUDA tensors of one device are needed, got "
                     f"{[str(t.device) for t in tensors if t is not None]}")


def refuse_dtypes(what, *tensors):
    raise TypeError(f"{what}: one dtype, float16 or bfloat16, got {[str(t.dtype) for t in tensors if t is not None]}")


def refuse_grad(what, hint=""):
    raise ValueError(f"{what}: an input requires a gradient, which this call does not record: call it under "
                     f"torch.no_grad(), or detach the input{hint}")


grad_enabled = torch.is_grad_enabled


def vector(t, dtype, n):
    """A contiguous 1-D tensor of n elements."""
    return t.dtype == dtype and t.shape == (n,) and t.is_contiguous()
