"""PyTorch front end over the C ABI: run a compiled module directly on ROCm tensors.

The reference's README suggests loading the dumped kernel "from PyTorch" (README.md:183); this is that hook.
`MonoNNFunction` wraps a loaded `MonoNNModule`: inputs and outputs are torch tensors on the GPU (no copies, the
launch goes onto torch's current stream), and the call is also registered as the custom operator
`mononn::forward(int handle, Tensor[] inputs) -> Tensor[]` so that it can sit inside a torch program or be A/B-timed
against `torch.nn.functional` on the same device.

torch is used for device memory and the stream only; all arithmetic happens in the generated HIP kernel.
"""
from __future__ import annotations

import ctypes
from typing import Dict, List, Sequence

import torch

from .binding import MonoNNModule

_TORCH_DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "s32": torch.int32, "s64": torch.int64, "pred": torch.bool,
                "u8": torch.uint8, "s8": torch.int8}
_REGISTRY: Dict[int, "MonoNNFunction"] = {}


class MonoNNFunction:
    """Callable view of a module whose constants are uploaded and which is loaded on `device`."""

    def __init__(self, module: MonoNNModule, outputs: Sequence[dict], device: int = 0, checked: bool = False):
        """`checked`: every call waits for its launch through mononn_module_synchronize and raises when a grid-barrier
        wait gave up (the outputs are then invalid).  Unchecked calls stay asynchronous on torch's current stream, and
        such a failure only shows in the caller's next MonoNNModule.synchronize()."""
        self.module = module
        self.checked = checked
        self.outputs = list(outputs)
        self.device = torch.device("cuda", device)
        info = module.buffer_info()
        self._param_bytes = info["parameters"]
        self._out_bytes = info["liveouts"]
        self._in_place = module.liveout_parameters()   # live-outs that are an input tensor, updated by the call
        self._updated = {i: _TORCH_DTYPE[t] for i, t in module.updated_parameters().items()}   # all such inputs, returned or not
        assert len(self._out_bytes) == len(self.outputs), "one {dtype, dims} entry per live-out is required"
        self._temp = None if module.owns_temp else torch.zeros(max(info["temp"], 256), dtype=torch.uint8, device=self.device)
        self._args_type = ctypes.c_void_p * (len(self._param_bytes) + len(self._out_bytes) + 1)
        self._temp_ptr = 0 if self._temp is None else self._temp.data_ptr()
        self._results = []   # extents, strides, type, parameter that is updated or -1
        for o, p, nbytes in zip(self.outputs, self._in_place, self._out_bytes):
            like = torch.empty(tuple(o["dims"]), dtype=_TORCH_DTYPE[o["dtype"]], device="meta")
            assert like.nbytes == nbytes
            assert p < 0 or like.dtype == self._updated[p], "a live-out that is an updated input has its declared type"
            self._results.append((tuple(like.shape), like.stride(), like.dtype, p))
        self.handle = id(self)
        _REGISTRY[self.handle] = self

    def close(self):
        _REGISTRY.pop(self.handle, None)

    def _input(self, i: int, t: torch.Tensor) -> torch.Tensor:
        """Parameter i from a tensor that is not simply the parameter's bytes: made contiguous, or refused."""
        assert t.is_cuda and t.device == self.device, "inputs must live on the module's GPU"
        assert t.is_contiguous() or i not in self._updated, "an input that the call updates in place must be contiguous"
        t = t.contiguous()
        nbytes = self._param_bytes[i]
        assert t.numel() * t.element_size() == nbytes, f"parameter needs {nbytes} bytes, got {t.numel() * t.element_size()}"
        assert t.data_ptr() % 16 == 0, "buffers must be 16-byte aligned"
        return t

    def __call__(self, *inputs: torch.Tensor) -> List[torch.Tensor]:
        # A call is a few microseconds of GPU work for the smallest modules, so the common case (tensors that can be
        # handed over as they are) does nothing twice.
        assert len(inputs) == len(self._param_bytes), f"expected {len(self._param_bytes)} tensors"
        device, held, ptrs = self.device, list(inputs), []
        for i, (t, nbytes) in enumerate(zip(inputs, self._param_bytes)):
            ptr = t.data_ptr()
            if ptr % 16 or t.nbytes != nbytes or t.device != device or not t.is_contiguous():
                held[i] = t = self._input(i, t)
                ptr = t.data_ptr()
            ptrs.append(ptr)
        if self._updated:
            recording, mine = torch.is_grad_enabled(), []
            for i, dtype in self._updated.items():
                t = held[i]
                mine.append(t)
                assert t.dtype == dtype, "an input that the call updates in place must have the declared type"
                assert ptrs.count(ptrs[i]) == 1, "an input that the call updates in place must not be passed twice"
                assert not (recording and t.requires_grad), "an input that the call updates in place must not require a gradient: the call records none"
        outs = []
        for dims, strides, dtype, param in self._results:
            if param >= 0:
                t = held[param]
                if t.shape != dims:
                    t = t.view(dims)
                ptrs.append(None)
            else:
                t = torch.empty_strided(dims, strides, dtype=dtype, device=device)   # a little cheaper than torch.empty
                ptrs.append(t.data_ptr())
            outs.append(t)
        ptrs.append(self._temp_ptr)
        args = self._args_type(*ptrs)   # the kernel's arguments, in order: parameters, live-outs, temp
        stream = torch._C._cuda_getCurrentRawStream(device.index)   # what torch.cuda.current_stream(device).cuda_stream says, without the stream object
        self.module.launch_arguments(args, stream)
        if self._updated:   # as torch's own in-place operations do: a backward pass that has saved such a tensor is to notice
            torch._C._increment_version(mine)   # what torch.autograd.graph.increment_version calls
        if self.checked:
            self.module.synchronize(stream)
        return outs


@torch.library.custom_op("mononn::forward", mutates_args=())
def _forward(handle: int, inputs: Sequence[torch.Tensor]) -> List[torch.Tensor]:
    fn = _REGISTRY[handle]
    # the operator is declared to change no input and to return new tensors
    assert not fn._updated, "a module that updates inputs in place is called through MonoNNFunction itself"
    return fn(*inputs)


@_forward.register_fake
def _(handle: int, inputs: Sequence[torch.Tensor]) -> List[torch.Tensor]:
    fn = _REGISTRY[handle]
    return [torch.empty(o["dims"], dtype=_TORCH_DTYPE[o["dtype"]], device=fn.device) for o in fn.outputs]


def forward(fn: MonoNNFunction, *inputs: torch.Tensor) -> List[torch.Tensor]:
    """torch.ops.mononn.forward on a MonoNNFunction."""
    return torch.ops.mononn.forward(fn.handle, list(inputs))
