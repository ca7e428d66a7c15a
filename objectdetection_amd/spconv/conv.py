"""spconv.SparseConv3d / SubMConv3d (call sites second/pytorch/models/middle.py:64-93,127-192,
second/pytorch/models/resnet.py:10-29).  Weight layout [kD,kH,kW,Cin,Cout], ``bias`` optional:
the state_dict keys and shapes match spconv 1.x so reference checkpoints load."""
import math

import torch
from torch import nn
from torch.nn import init

from .. import ops
from .modules import SparseModule
from .tensor import SparseConvTensor


def _ntuple(v, n):
    if isinstance(v, (list, tuple)):
        v = [int(x) for x in v]
        if len(v) != n:
            raise ValueError(f"expected {n} values, got {v}")
        return v
    return [int(v)] * n


class SparseConvolution(SparseModule):
    def __init__(self, ndim, in_channels, out_channels, kernel_size=3, stride=1, padding=0,
                 dilation=1, groups=1, bias=True, subm=False, output_padding=0,
                 transposed=False, inverse=False, indice_key=None, fused_bn=False):
        super().__init__()
        assert groups == 1, "spconv only supports groups == 1"
        if transposed or inverse:
            raise NotImplementedError(
                "transposed / inverse sparse convolutions are not on the SECOND front-end path")
        if ndim not in (2, 3):
            raise NotImplementedError("only 2-D and 3-D sparse convolutions are supported")
        self.ndim = ndim
        self.in_channels = in_channels
        self.out_channels = out_channels
        self.kernel_size = _ntuple(kernel_size, ndim)
        self.conv1x1 = all(k == 1 for k in self.kernel_size)
        self.stride = _ntuple(stride, ndim)
        self.padding = _ntuple(padding, ndim)
        self.dilation = _ntuple(dilation, ndim)
        self.output_padding = _ntuple(output_padding, ndim)
        self.transposed = transposed
        self.inverse = inverse
        self.groups = groups
        self.subm = subm
        self.indice_key = indice_key
        self.fused_bn = fused_bn
        for s, d in zip(self.stride, self.dilation):
            assert s == 1 or d == 1, "don't support stride > 1 together with dilation > 1"
        self.weight = nn.Parameter(torch.Tensor(*self.kernel_size, in_channels, out_channels))
        if bias:
            self.bias = nn.Parameter(torch.Tensor(out_channels))
        else:
            self.register_parameter("bias", None)
        self.reset_parameters()

    def reset_parameters(self):
        init.kaiming_uniform_(self.weight, a=math.sqrt(5))
        if self.bias is not None:
            fan_in, _ = init._calculate_fan_in_and_fan_out(self.weight)
            bound = 1 / math.sqrt(fan_in)
            init.uniform_(self.bias, -bound, bound)

    def extra_repr(self):
        return (f"{self.in_channels}, {self.out_channels}, kernel_size={self.kernel_size}, "
                f"stride={self.stride}, padding={self.padding}, dilation={self.dilation}, "
                f"subm={self.subm}, indice_key={self.indice_key}")

    def _as3(self, v, fill):
        return list(v) if self.ndim == 3 else [fill] + list(v)

    def get_rulebook(self, input):
        """Rulebook for this layer on ``input``: cached per ``indice_key`` in
        ``input.indice_dict`` exactly as spconv does (key None is never cached)."""
        rb = input.find_indice_pair(self.indice_key)
        if rb is not None:
            if self.subm and not (isinstance(rb, ops.Rulebook) and rb.subm):
                rb = None
            elif rb.ksize != self._as3(self.kernel_size, 1):
                raise ValueError(
                    f"indice_key {self.indice_key!r} reused with a different kernel size")
        if rb is None:
            shape = input.spatial_shape if self.ndim == 3 else [1] + list(input.spatial_shape)
            indices = input.indices
            if indices.dtype != torch.int32:
                indices = indices.int()
            if self.ndim == 2:  # (b,y,x) -> (b,0,y,x)
                z = torch.zeros_like(indices[:, :1])
                indices = torch.cat([indices[:, :1], z, indices[:, 1:]], dim=1)
            rb = ops.build_rulebook(indices, input.batch_size, shape,
                                    self._as3(self.kernel_size, 1), self._as3(self.stride, 1),
                                    self._as3(self.padding, 0), self._as3(self.dilation, 1),
                                    self.subm)
            if self.indice_key is not None:
                input.indice_dict[self.indice_key] = rb
        return rb

    def forward(self, input, _scale=None, _shift=None, _relu=False, _f8=None):
        assert isinstance(input, SparseConvTensor)
        features = input.features
        if not features.is_cuda:
            raise RuntimeError("spconv (objectdetection_amd) runs on the GPU only: no CPU path")
        if self.pointwise:
            # spconv 1.x's short cut for an all-ones kernel (SparseConvolution.forward; used by
            # second/pytorch/models/resnet.py:20-29,69-110): a plain row-wise GEMM, no rulebook --
            # a library GEMM, so any channel count (SparseBottleneck's 256) goes through; under
            # ops.conv_math("f8") the product on 8-bit rows with its fused epilogue
            w = self.weight.view(self.in_channels, self.out_channels)
            if ops.get_conv_math() == "f8":
                out = self._pointwise_f8(features, w, _scale, _shift, _relu, _f8)
            else:
                out = torch.mm(features, w.to(features.dtype))
                if self.bias is not None:
                    out = out + self.bias.to(out.dtype)
                if _scale is not None:
                    out = out * _scale.to(out.dtype)
                if _shift is not None:
                    out = out + _shift.to(out.dtype)
                if _relu:
                    out = torch.relu(out)
            out_tensor = SparseConvTensor(out, input.indices, input.spatial_shape,
                                          input.batch_size)
            out_tensor.indice_dict = input.indice_dict
            out_tensor.grid = input.grid
            return out_tensor
        rb = self.get_rulebook(input)
        if self.ndim == 3:
            out_indices, out_shape = rb.out_indices, rb.out_shape
        else:
            out_indices = rb.out_indices[:, [0, 2, 3]].contiguous()
            out_shape = rb.out_shape[1:]
        fused = _scale is not None or _shift is not None or _relu
        if fused:
            # inference epilogue fusion (SparseSequential): conv (+bias) -> affine -> relu
            shift = _shift
            if self.bias is not None:
                b = self.bias.float()
                shift = b * _scale + _shift if _scale is not None else (
                    b + _shift if _shift is not None else b)
            x = features if features.dtype == torch.float32 else features.float()
            out = self._inference_forward(x, rb, _scale,
                                          None if shift is None else shift.contiguous(), _relu)
            out = out.to(features.dtype)
        elif not torch.is_grad_enabled():
            x = features if features.dtype == torch.float32 else features.float()
            shift = None if self.bias is None else self.bias.float().contiguous()
            out = self._inference_forward(x, rb, None, shift, False)
            out = out.to(features.dtype)
        else:
            out = ops.indice_conv(features, self.weight, rb)
            if self.bias is not None:
                out = out + self.bias
        out_tensor = SparseConvTensor(out, out_indices, out_shape, input.batch_size)
        out_tensor.indice_dict = input.indice_dict
        out_tensor.grid = input.grid
        return out_tensor

    @property
    def pointwise(self):
        """A row-wise linear layer: no rulebook, no neighbours."""
        return self.conv1x1 and all(st == 1 for st in self.stride)

    def _pointwise_f8(self, x, w, scale, shift, relu, f8):
        """Rows x [K, Cin] (or, in inference, their 8-bit form ``f8`` already) through w [Cin, Cout]
        on 8-bit operands."""
        if torch.is_grad_enabled() and (x.requires_grad or self.weight.requires_grad or (
                self.bias is not None and self.bias.requires_grad)):
            out = ops.f8_linear(x, w, self.bias, turned=True)
            return torch.relu(out) if relu else out
        if self.bias is not None:
            b = self.bias.detach().float()
            b = b if scale is None else b * scale
            shift = b if shift is None else b + shift
        scale = None if scale is None else scale.float().contiguous()
        shift = None if shift is None else shift.float().contiguous()
        if f8 is None:
            return ops.f8_product(x, self._weight_image("f8"), scale, shift, relu)
        return ops.f8_matmul(f8, self._weight_image("f8"), scale, shift, relu, out_dtype=x.dtype)

    def _inference_forward(self, x, rb, scale, shift, relu):
        """No-grad forward: fp32 MFMA, or -- under ``ops.conv_math("bf16x3")`` and for 32 / 64 /
        128 channels on both sides -- split bf16 operands at fp32 tolerance (include/lcf.h)."""
        cin, cout = self.in_channels, self.out_channels
        mode = ops.get_conv_math()
        if mode in ("bf16x3", "bf16x8") and ops.bf16_supported(cin, cout):
            planes = 3 if mode == "bf16x8" else 2
            return ops.conv_forward_bf16x3(x, self._weight_image(planes), rb.out_nbr, rb.k_out,
                                           rb.kvol, cin, cout, scale, shift, relu, planes=planes)
        return ops.conv_forward(x, self._weight_image(), rb.out_nbr, rb.k_out, rb.kvol, cin, cout,
                                scale, shift, relu)

    def __getstate__(self):  # copies and pickles make their own images
        return {k: v for k, v in self.__dict__.items() if not k.startswith("_wimg")}

    def _weight_image(self, planes=0):
        """MFMA weight image (planes 2 / 3: the split bf16x3 / bf16x8 image; "f8": a pointwise conv's
        8-bit form), cached until the parameter is modified in place or replaced.  The cache holds the
        values that it was made from, so that their address stays theirs, and an event, for users on
        another stream.  In a graph's capture the image is always made, whether one is cached or not:
        it is then the graph's own memory, and replays follow the weight (a cached image would be freed
        under the graph by the next call with a changed weight)."""
        w = self.weight
        if torch.cuda.is_current_stream_capturing():
            return self._make_weight_image(planes)
        tag = (w.data_ptr(), w._version, w.device, w.dtype)
        name = f"_wimg{planes}"
        cache = getattr(self, name, None)
        if cache is None or cache[0] != tag:
            img = self._make_weight_image(planes)
            maker = torch.cuda.current_stream(w.device)
            cache = (tag, img, w.detach(), maker, maker.record_event())
            object.__setattr__(self, name, cache)
        else:
            user = torch.cuda.current_stream(w.device)
            if user != cache[3]:
                user.wait_event(cache[4])
                for t in cache[1] if isinstance(cache[1], tuple) else (cache[1],):
                    t.record_stream(user)
        return cache[1]

    def _make_weight_image(self, planes):
        w = self.weight
        if planes == "f8":
            return ops.f8_weight_image(w.view(self.in_channels, self.out_channels), transpose=True)
        return ops.weight_image_bf16x3(w, planes=planes) if planes else ops.weight_image(w)


class SparseConv2d(SparseConvolution):
    def __init__(self, in_channels, out_channels, kernel_size, stride=1, padding=0, dilation=1,
                 groups=1, bias=True, indice_key=None):
        super().__init__(2, in_channels, out_channels, kernel_size, stride, padding, dilation,
                         groups, bias, indice_key=indice_key)


class SparseConv3d(SparseConvolution):
    def __init__(self, in_channels, out_channels, kernel_size, stride=1, padding=0, dilation=1,
                 groups=1, bias=True, indice_key=None):
        super().__init__(3, in_channels, out_channels, kernel_size, stride, padding, dilation,
                         groups, bias, indice_key=indice_key)


class SubMConv2d(SparseConvolution):
    def __init__(self, in_channels, out_channels, kernel_size, stride=1, padding=0, dilation=1,
                 groups=1, bias=True, indice_key=None):
        super().__init__(2, in_channels, out_channels, kernel_size, stride, padding, dilation,
                         groups, bias, True, indice_key=indice_key)


class SubMConv3d(SparseConvolution):
    def __init__(self, in_channels, out_channels, kernel_size, stride=1, padding=0, dilation=1,
                 groups=1, bias=True, indice_key=None):
        super().__init__(3, in_channels, out_channels, kernel_size, stride, padding, dilation,
                         groups, bias, True, indice_key=indice_key)
