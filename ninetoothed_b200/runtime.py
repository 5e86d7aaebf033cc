"""Launch runtime of the B200 backend: argument binding, validation and errors.

Mirrors the reference runtime's contract for a materialized kernel
(src/ninetoothed/compiler/runtime.py):

- `KernelLaunchError` (runtime.py:31-35) is raised for a nonzero return code;
- public arguments are bound positionally or by keyword and checked for count,
  duplicates, unknown names and missing names with the same `TypeError`
  messages as `_public_values` (runtime.py:1147-1185);
- tensors are checked for rank, device type and a single common device
  (`_validate_tensor_contract`, runtime.py:1218-1264);
- an output with zero elements launches nothing and is returned as is
  (`_empty_launch`, runtime.py:1411-1422);
- the call returns the first output (`_first_output`, runtime.py:1397-1398);
- kernels run on the caller's current CUDA stream of the tensors' device
  (materializers/cuda.py:122-123).
"""

from dataclasses import dataclass, field
from typing import Any, Callable

import torch

from ninetoothed_b200 import _lib


class KernelLaunchError(RuntimeError):
    """Raised when a materialized backend launcher reports an error."""

    def __init__(self, error_code):
        self.error_code = error_code
        super().__init__(f"Kernel launch failed with error code: {error_code}.")


FLOAT_DTYPES = (torch.float16, torch.bfloat16, torch.float32)
HALF_DTYPES = (torch.float16, torch.bfloat16)
FP8_DTYPES = tuple(getattr(torch, name) for name in ("float8_e4m3fn", "float8_e5m2") if hasattr(torch, name))
GEMM_DTYPES = HALF_DTYPES + FP8_DTYPES + (torch.float32,)


_DTYPE_CODES = {getattr(torch, name): code for name, code in _lib.DTYPE_CODES.items() if hasattr(torch, name)}


def dtype_code(dtype: torch.dtype) -> int:
    return _DTYPE_CODES[dtype]


@dataclass(frozen=True)
class TensorArg:
    """Contract of one tensor argument: its rank and the dtypes the kernel takes.
    An optional argument may be None."""

    name: str
    ndim: int
    dtypes: tuple = FLOAT_DTYPES
    optional: bool = False


@dataclass(frozen=True)
class ScalarArg:
    name: str


@dataclass
class Kernel:
    """A callable kernel with the reference's `make()` calling convention.

    `kernel(*args, **meta)` binds the public arguments (`args`) and meta
    keywords (`meta`), validates them, launches on the current stream and
    returns the first output.
    """

    name: str
    args: tuple
    outputs: tuple
    launch: Callable[[dict, int], int]
    meta: tuple = ()
    meta_defaults: dict = field(default_factory=dict)

    def __post_init__(self):
        # what every call looks up, once
        self.public_args = tuple(arg.name for arg in self.args)
        self._tensor_args = tuple(
            (arg.name, arg.ndim, frozenset(arg.dtypes), arg) for arg in self.args if isinstance(arg, TensorArg)
        )
        self._accepted = frozenset(self.public_args) | frozenset(self.meta)
        self._required = self.public_args + tuple(self.meta)

    def __call__(self, *args, **kwargs):
        values = self._public_values(args, kwargs)
        device = self._validate(values)
        output = values[self.outputs[0]] if self.outputs else None
        for name in self.outputs:
            if values[name].numel() == 0:
                return output
        if device.index == torch.cuda.current_device():
            code = self.launch(values, current_raw_stream(device.index))
        else:
            with torch.cuda.device(device):
                code = self.launch(values, current_raw_stream(device.index))
        if code != 0:
            raise KernelLaunchError(code)
        return output

    # ------------------------------------------------------------- binding
    def _public_values(self, args, kwargs) -> dict[str, Any]:
        public = self.public_args
        if len(args) > len(public):
            raise TypeError(f"Expected at most {len(public)} arguments.")
        if kwargs:
            duplicates = tuple(name for name in kwargs if name in public and public.index(name) < len(args))
            if duplicates:
                raise TypeError(f"Kernel arguments passed twice: {', '.join(sorted(duplicates))}.")
            if not self._accepted.issuperset(kwargs):
                unknown = tuple(name for name in kwargs if name not in self._accepted)
                raise TypeError(f"Unknown kernel arguments: {', '.join(sorted(unknown))}.")
        values = dict(self.meta_defaults)
        values.update(zip(public, args))
        values.update(kwargs)
        if len(values) < len(self._required):
            missing = tuple(name for name in self._required if name not in values)
            raise TypeError(f"Missing kernel arguments: {', '.join(missing)}.")
        return values

    def _validate(self, values) -> torch.device:
        device = None
        for name, ndim, dtypes, arg in self._tensor_args:
            value = values[name]
            if value is None and arg.optional:
                continue
            if not isinstance(value, torch.Tensor):
                raise TypeError(f"Kernel argument `{name}` must be a tensor.")
            if value.dim() != ndim:
                raise TypeError(f"Kernel argument `{name}` has rank {value.dim()}; expected {ndim}.")
            if value.device != device:
                if value.device.type != "cuda":
                    raise TypeError(f"Kernel argument `{name}` must be on a CUDA device.")
                if device is not None:
                    raise TypeError("All tensor arguments must use the same CUDA device.")
                device = value.device
            if value.dtype not in dtypes:
                expected = ", ".join(str(d).split(".")[-1] for d in arg.dtypes)
                raise TypeError(
                    f"Kernel argument `{name}` has dtype {str(value.dtype).split('.')[-1]}; "
                    f"expected one of {expected}."
                )
        if device is None:
            raise TypeError("Kernel call has no tensor arguments.")
        return device


def _public_raw_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# The caller's current CUDA stream on a device, as an address.  torch's own
# lookup of it takes a tenth of the time of building a Stream object.
current_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _public_raw_stream)


def ptr(tensor: torch.Tensor) -> int:
    return tensor.data_ptr()


def check_same_dtype(values, names):
    dtype = values[names[0]].dtype
    for name in names:
        if values[name].dtype != dtype:
            listing = ", ".join(f"`{name}`" for name in names)
            raise TypeError(f"Kernel arguments {listing} must share one dtype.")


def device_status(stream: int = None) -> int:
    """Synchronise `stream` and return (and clear) the library's device error word."""
    import ctypes

    if stream is None:
        stream = torch.cuda.current_stream().cuda_stream
    status = ctypes.c_int(0)
    code = _lib.library().nt_b200_device_status(stream, ctypes.byref(status))
    if code != 0:
        raise KernelLaunchError(code)
    return status.value
