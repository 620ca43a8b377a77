"""Quantized Linear / MLP layers: the caller side of q_gemm_dequant.

Mirror of the C++ classes in include/mlxr_linear.h, which follow the reference's
core/graph/layers.h:59-94 (Linear: in_features, out_features, bias; forward(x) over
x [..., in_features] with M = batch * seq, layers.cpp:86-99) and MLP::forward
(layers.cpp:391-414: down(swish(gate(x)) * up(x))).  Weights are packed GGUF blocks on the
device, or 8-bit floats with a scale for each 128 x 128 (Fp8Weight); every computation runs in
libmlxr_qgemm.so (torch supplies memory and streams).
"""
from . import fp8, qgemm
from .fp8 import Fp8Rows, Fp8Weight
from .qgemm import BF16, F16, F32, PackedWeight, QGemmError


def _dt(torch, dtype):
    return {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}[dtype]


def swiglu(gate, up, out=None, stream=None):
    """swish(gate) * up elementwise (mlxr_swiglu), in the dtype of gate."""
    torch = qgemm._torch()
    if gate.shape != up.shape or gate.dtype != up.dtype:
        raise QGemmError(-3, "gate and up must have the same shape and dtype")
    gate, up = gate.contiguous(), up.contiguous()
    out = torch.empty_like(gate) if out is None else out
    qgemm._check(qgemm.lib().mlxr_swiglu(gate.data_ptr(), up.data_ptr(), out.data_ptr(), gate.numel(), _dt(torch, gate.dtype),
                   qgemm._stream_ptr(stream)))
    return out


class Linear:
    """y = x W^T (+ b) with W [out_features, in_features] held as packed GGUF blocks or as an ``Fp8Weight``."""

    def __init__(self, in_features, out_features, bias=False):
        if in_features <= 0 or out_features <= 0:
            raise QGemmError(-1, "Linear: features must be positive")
        self.in_features, self.out_features, self.has_bias = in_features, out_features, bias
        self.weight = None
        self.bias = None

    def load_weight(self, src, quant_type=None, name=None, device="cuda"):
        """src: GGUF block bytes (numpy/torch uint8) with quant_type, a PackedWeight, an Fp8Weight, or a
        GGUFFile with the tensor name."""
        from .gguf import GGUFFile
        if isinstance(src, (PackedWeight, Fp8Weight)):
            pw = src
        elif isinstance(src, GGUFFile):
            info = src.find_tensor(name)
            if info is None:
                raise QGemmError(-1, f"GGUF tensor not found: {name}")
            if info.dimensions != [self.in_features, self.out_features]:
                raise QGemmError(-3, f"GGUF tensor {name} does not have dims {{in_features, out_features}}")
            pw = src.upload(name, device=device)
        else:
            pw = qgemm.pack_weights(src, self.out_features, self.in_features, quant_type, device=device)
        if (pw.N, pw.K) != (self.out_features, self.in_features):
            raise QGemmError(-3, "weight shape does not match [out_features, in_features]")
        self.weight = pw
        return self

    def set_bias(self, bias):
        if not self.has_bias:
            raise QGemmError(-1, "Linear was built without bias")
        if bias.dim() != 1 or bias.shape[0] != self.out_features:
            raise QGemmError(-3, "Bias shape must be [N]")
        self.bias = bias

    def forward(self, x, stream=None, lora=None, adapter_ids=None):
        """x W^T (+ b); with ``lora`` (a LoraBank of this layer's shape) and ``adapter_ids`` [tokens] (int32,
        -1: none) also each token's own adapter (lora_apply).  An 8-bit weight also takes x as ``Fp8Rows`` [M, in_features]
        (rms_norm's), giving bfloat16, without adapters; other x it rounds to 8 bits first."""
        if stream is not None:  # copies of rows that lie apart and intermediate results are that stream's too
            with qgemm._torch().cuda.stream(stream):
                return self.forward(x, lora=lora, adapter_ids=adapter_ids)
        if self.weight is None:
            raise QGemmError(-1, "Linear: weight not loaded")
        if (lora is None) != (adapter_ids is None):
            raise QGemmError(-1, "Linear: lora and adapter_ids go together")
        if lora is not None and (lora.N, lora.K) != (self.out_features, self.in_features):
            raise QGemmError(-3, "adapters do not match [out_features, in_features]")
        if self.has_bias and self.bias is None:
            raise QGemmError(-1, "Linear: bias not set")
        eight = isinstance(self.weight, Fp8Weight)
        if isinstance(x, Fp8Rows):
            if not eight or lora is not None:
                raise QGemmError(-1, "Linear: rows in 8 bits need an 8-bit weight and take no adapters")
            return fp8.fp8_matmul(x, self.weight, bias=self.bias)
        if x.dim() < 1 or x.shape[-1] != self.in_features:
            raise QGemmError(-3, "Input shape must be [..., in_features]")
        lead = x.shape[:-1]
        M = 1
        for d in lead:
            M *= int(d)
        x2 = x.reshape(M, self.in_features)
        if eight:
            y = fp8.fp8_matmul(x2, self.weight, bias=self.bias)
        else:
            y = qgemm.q_gemm_dequant(x2, self.weight, M, self.out_features, self.in_features, self.weight.qtype,
                                     bias=self.bias)
        if lora is not None:
            y = lora.apply(x2, adapter_ids, y, out=y)
        return y.reshape(*lead, self.out_features)

    __call__ = forward


class MLP:
    """down(swish(gate(x)) * up(x)) through mlxr_qgemm_mlp: at M = 1 the whole block is one
    launch; above, the fused gate/up/gating launch and the down projection.  The layer holds
    the workspace (sync words, h, split-K partials).  With 8-bit weights (Fp8Weight) x is rounded to 8 bits once
    for gate and up, or comes as ``Fp8Rows``, and the gated rows once for down.  Projections built with a bias
    are run one by one."""

    def __init__(self, hidden_size, intermediate_size):
        self.hidden_size, self.intermediate_size = hidden_size, intermediate_size
        self.gate_proj = Linear(hidden_size, intermediate_size)
        self.up_proj = Linear(hidden_size, intermediate_size)
        self.down_proj = Linear(intermediate_size, hidden_size)
        self._ws = None

    def forward(self, x, stream=None):
        if stream is not None:  # as in Linear
            with qgemm._torch().cuda.stream(stream):
                return self.forward(x)
        gw, uw, dw = self.gate_proj.weight, self.up_proj.weight, self.down_proj.weight
        rows = isinstance(x, Fp8Rows)
        if not rows and (x.dim() < 1 or x.shape[-1] != self.hidden_size):
            raise QGemmError(-3, "Input shape must be [..., hidden_size]")
        if gw is None or uw is None or dw is None:
            raise QGemmError(-1, "MLP: weights not loaded")
        if rows or isinstance(gw, Fp8Weight) or isinstance(uw, Fp8Weight) or isinstance(dw, Fp8Weight):
            return self._forward8(x, rows)
        lead = x.shape[:-1]
        x2 = x.reshape(-1, self.hidden_size)
        biases = self.gate_proj.has_bias or self.up_proj.has_bias or self.down_proj.has_bias
        if (gw.qtype, gw.N) == (uw.qtype, uw.N) and not biases:
            if self._ws is None:
                self._ws = qgemm.MlpWorkspace(x.device)
            y = qgemm.q_gemm_mlp(x2, gw, uw, dw, self._ws)
        else:
            g = self.gate_proj.forward(x2)
            u = self.up_proj.forward(x2)
            h = swiglu(g, u, out=g)
            y = self.down_proj.forward(h)
        return y.reshape(*lead, self.hidden_size)

    def _forward8(self, x, rows):
        """forward where at least one weight is 8-bit, or x is Fp8Rows."""
        gate, up = self.gate_proj, self.up_proj
        both = isinstance(gate.weight, Fp8Weight) and isinstance(up.weight, Fp8Weight)
        if rows and not both:
            raise QGemmError(-1, "MLP: rows in 8 bits need 8-bit gate and up weights")
        if both:
            lead, dtype = ((x.data.shape[0],), None) if rows else (x.shape[:-1], x.dtype)
            if any(p.has_bias and p.bias is None for p in (gate, up)):
                raise QGemmError(-1, "MLP: bias not set")
            x8 = x if rows else fp8.quantize_fp8(x)
            g, u = (fp8.fp8_matmul(x8, p.weight, bias=p.bias, out_dtype=dtype) for p in (gate, up))
        else:
            lead, x2 = x.shape[:-1], x.reshape(-1, self.hidden_size)
            g, u = gate.forward(x2), up.forward(x2)
        h = swiglu(g, u, out=g)
        return self.down_proj.forward(h).reshape(*lead, self.hidden_size)

    __call__ = forward
