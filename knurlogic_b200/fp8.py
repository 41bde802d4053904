"""Block-scaled e4m3 products and products of rows grouped by expert.

* `quantize_fp8(x)`: bf16 rows -> e4m3 values and a float32 scale for each
  row and 128 inputs;
* `Fp8Linear(weight, weight_scale_inv)`: a dense linear with e4m3 weights and
  a float32 scale for each 128 x 128 block, its inputs quantized on the way in
  (the experts' form is `Fp8SwitchLinear`);
* `grouped_linear(x, weight, offsets)`: rows in expert order, ragged counts
  in a device tensor, times their expert's weights (bf16 or e4m3).

Every call runs on the tensor's device and its current stream, allocates its
workspace from torch's caching allocator and does not synchronise. The
reference has no counterpart: these serve checkpoints in the block-scaled
format next to its VQ artifacts.
"""
from __future__ import annotations

import torch
from torch import nn

from . import _lib
from .switch_layers import Fp8Buffers, _contig, call_on, check_fp8_weight, fp8_descriptor, require_cuda

GROUP = 128
_status: dict = {}


def _status_word(device: torch.device) -> torch.Tensor | None:
    """The device's word that a bounded wait raises when it runs out. None
    inside a stream capture that no call and no module on the device came
    before (a word made there would be the graph's own)."""
    w = _status.get(device.index)
    if w is None and not torch.cuda.is_current_stream_capturing():
        with torch.inference_mode(False):                    # cleared in any mode later
            w = torch.zeros(1, dtype=torch.int32, device=device)
        torch.cuda.current_stream(device).synchronize()      # zero before another stream's kernels see it
        w = _status.setdefault(device.index, w)
    return w


def check_status(device=None) -> None:
    """Raise `TimeoutError` when a bounded device wait of `Fp8Linear` or
    `grouped_linear` ran out on `device` since the last check: an output since
    then is wrong. Synchronises with the device."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    w = _status.get(dev.index if dev.index is not None else torch.cuda.current_device())
    if w is not None:
        torch.cuda.synchronize(w.device)
        if int(w.item()):
            w.zero_()
            raise TimeoutError("a bounded device wait ran out in an e4m3 or grouped product")


def _rows(x: torch.Tensor, features: int) -> torch.Tensor:
    """x as [rows, features] bf16 with unit stride along a row; a copy only
    where a row's pitch or start is not the kernels' (16 bytes)."""
    if not x.is_cuda:
        require_cuda(x)
    if x.dtype is not torch.bfloat16:
        raise TypeError(f"x must be bfloat16, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] != features:
        raise ValueError(f"x {tuple(x.shape)} has not {features} features")
    if x.dim() != 2:
        x = x.reshape(-1, features)
    pitch, one = x.stride()
    if x.shape[0] and (one != 1 or pitch < features or pitch % 8 or x.data_ptr() % 16):
        x = x.contiguous() if not x.is_contiguous() else x.clone()
    return x


def _pitch(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def quantize_fp8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., K] bf16 -> (q [..., K] float8_e4m3fn, scales [..., ceil(K/128)]
    float32), x ~ q * scale. Of a row's group of 128 inputs (the last one
    ragged) with the largest magnitude a, at least 2^-100:
        scale = f32(a / 448),  q = e4m3(448 x / a)
    -- the exact quotient rounded once, ties to even. A NaN or an infinity in
    a group makes its scale NaN. K is a multiple of 16."""
    K = x.shape[-1] if x.dim() else 0
    if K <= 0 or K % 16:
        raise ValueError(f"x {tuple(x.shape)}: the last dimension must be a multiple of 16")
    xr = _rows(x, K)
    q = (torch.empty_like(x, dtype=torch.float8_e4m3fn) if x.is_contiguous()
         else x.new_empty(x.shape, dtype=torch.float8_e4m3fn))
    s = x.new_empty((*x.shape[:-1], -(-K // GROUP)), dtype=torch.float32)
    if xr.shape[0]:
        call_on(x.device, "vqmoe_quantize_fp8", xr.data_ptr(), xr.shape[0], K, _pitch(xr), q.data_ptr(), s.data_ptr())
    return q, s


def _run(d: _lib.Linear, x: torch.Tensor, offsets, out: torch.Tensor) -> torch.Tensor:
    """`vqmoe_grouped_linear` of rows x [P, K] into out [P, N]."""
    P = x.shape[0]
    if P == 0:
        return out
    dev = x.device
    n = _lib.lib().vqmoe_grouped_linear_workspace_size(d, P)
    ws = x.new_empty(n, dtype=torch.uint8) if n else None
    st = _status.get(dev.index)
    if st is None:
        st = _status_word(dev)
    call_on(dev, "vqmoe_grouped_linear", d, x.data_ptr(), P, _pitch(x),
             offsets.data_ptr() if offsets is not None else None, out.data_ptr(),
             _lib.OUT_F32 if out.dtype is torch.float32 else _lib.OUT_BF16,
             ws.data_ptr() if n else None, n, st.data_ptr() if st is not None else None)
    return out


def _same_device(x: torch.Tensor, **others: torch.Tensor) -> None:
    for name, t in others.items():
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")


class Fp8Linear(Fp8Buffers, nn.Module):
    """y = x W^T with block-scaled e4m3 weights: `weight [OUT, IN]`
    float8_e4m3fn, `weight_scale_inv [ceil(OUT/128), ceil(IN/128)]` (float32,
    or bf16 widened). OUT and IN are multiples of 16.

    `forward(x [..., IN] bf16, out_dtype=torch.bfloat16)`: the rows are
    quantized (`quantize_fp8`), the products summed in float32 with both
    scales applied to each block's sum, and rounded once to bf16 (or kept as
    float32, for logits). The order of a row's float32 additions goes by the
    number of rows in the call, never by their values."""

    weight_dims = 2

    def __init__(self, weight: torch.Tensor, weight_scale_inv: torch.Tensor):
        super().__init__()
        check_fp8_weight(weight, weight_scale_inv, 2)
        self.register_buffer("weight", weight.contiguous())
        self.register_buffer("weight_scale_inv", weight_scale_inv.to(torch.float32).contiguous())
        self._report()

    def _report(self) -> None:
        """The device has its status word before the module's first call,
        which may be captured."""
        if self.weight.is_cuda:
            _status_word(self.weight.device)

    def _apply(self, *args, **kwargs):
        r = super()._apply(*args, **kwargs)
        self._report()
        return r

    @property
    def out_features(self):
        return self.weight.shape[0]

    @property
    def in_features(self):
        return self.weight.shape[1]

    def descriptor(self) -> _lib.Linear:
        w = self.weight
        require_cuda(w, self.weight_scale_inv)
        return fp8_descriptor(self)

    def forward(self, x: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        if out_dtype not in (torch.bfloat16, torch.float32):
            raise TypeError(f"out_dtype {out_dtype} (bfloat16 or float32)")
        w = self._buffers["weight"]
        N, K = w.shape
        xr = _rows(x, K)
        if w.device != x.device:
            _same_device(x, weight=w)
        out = x.new_empty((*x.shape[:-1], N), dtype=out_dtype)
        return _run(fp8_descriptor(self), xr, None, out)


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor,
                   weight_scale_inv: torch.Tensor | None = None, out: torch.Tensor | None = None,
                   out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """out[r] = x[r] weight[e]^T for offsets[e] <= r < offsets[e + 1]: rows in
    expert order, any number of them an expert (none included).

    x [P, IN] bf16 (rows may lie at a pitch); weight [E, OUT, IN] bf16, or
    float8_e4m3fn with `weight_scale_inv [E, ceil(OUT/128), ceil(IN/128)]`
    float32 (x is then quantized as by `quantize_fp8`); offsets [E + 1] int32
    on the device, ascending (not read on the host: values outside [0, P] are
    clamped, one below an earlier offset counts as the largest before it);
    E <= 1024, OUT and IN multiples of 16. Sums are float32, rounded once to
    `out_dtype` (bf16 or float32). Rows that lie in no
    group -- before the first offset or behind the last -- are left as they
    were in `out` (contiguous [P, OUT]); without `out` they are unset."""
    require_cuda(x, weight, offsets, weight_scale_inv, out)
    if x.dim() != 2:
        raise ValueError(f"x must be [rows, IN], got {tuple(x.shape)}")
    if weight_scale_inv is not None:
        check_fp8_weight(weight, weight_scale_inv, 3)
        if weight_scale_inv.dtype != torch.float32:
            raise TypeError(f"weight_scale_inv must be float32, got {weight_scale_inv.dtype}")
    elif weight.dim() != 3 or weight.dtype != torch.bfloat16:
        raise ValueError(f"weight must be [E, OUT, IN] bfloat16 (or float8_e4m3fn with weight_scale_inv), got "
                         f"{tuple(weight.shape)} {weight.dtype}")
    E, N, K = weight.shape
    if 0 in weight.shape or N % 16 or K % 16:
        raise ValueError(f"weight {tuple(weight.shape)}: OUT and IN must be multiples of 16")
    if E > 1024:
        raise ValueError(f"{E} experts (at most 1024)")
    if offsets.dtype != torch.int32 or tuple(offsets.shape) != (E + 1,):
        raise ValueError(f"offsets must be [{E + 1}] int32, got {tuple(offsets.shape)} {offsets.dtype}")
    if out is None:
        if out_dtype not in (torch.bfloat16, torch.float32):
            raise TypeError(f"out_dtype {out_dtype} (bfloat16 or float32)")
        out = x.new_empty((x.shape[0], N), dtype=out_dtype)
    elif (tuple(out.shape) != (x.shape[0], N) or out.dtype not in (torch.bfloat16, torch.float32)
          or not out.is_contiguous()):
        raise ValueError(f"out must be contiguous [{x.shape[0]}, {N}] bfloat16 or float32, got {tuple(out.shape)} "
                         f"{out.dtype}")
    _same_device(x, weight=weight, offsets=offsets, out=out)
    xr = _rows(x, K)
    w, off = _contig(weight), _contig(offsets)
    d = _lib.Linear(format=_lib.FMT_DENSE_BF16, num_experts=E, out_features=N, in_features=K, weight=w.data_ptr())
    if weight_scale_inv is not None:
        _same_device(x, weight_scale_inv=weight_scale_inv)
        ws = _contig(weight_scale_inv)
        d.format, d.scales, d.group_size = _lib.FMT_FP8_BLOCK, ws.data_ptr(), GROUP
    return _run(d, xr, off, out)
