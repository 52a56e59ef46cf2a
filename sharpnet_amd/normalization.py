"""Host side of the norms before and after a block (the layer and RMS norms of Prod/GPU/Kernels/SinglePrecision.cu:32-284
fused with the residual connection around a block) on GPUTensor.

``u = x + residualScale * act(gate) * N_post(y)`` and ``h = N_pre(u)``, forward and backward, each in one pass over the rows
in libsharpnet_hip.so.  x is the residual stream, y the output of the block behind it (MultiheadAttention, Linear ...), h
what the next block reads.
"""
import ctypes

from .gpu_tensor import GPUTensor
from .hiplib import (ACT_NONE, ACT_SIGMOID, ACT_TANH, BlockNormDesc, NORM_LAYER, NORM_NONE, NORM_RMS, SharpNetHipError, CublasStatus,
                     TYPES, check_status)

_NORMS = {None: NORM_NONE, "none": NORM_NONE, "rms": NORM_RMS, "layer": NORM_LAYER}
_GATES = {None: ACT_NONE, "none": ACT_NONE, "sigmoid": ACT_SIGMOID, "tanh": ACT_TANH,
          "CUDNN_ACTIVATION_IDENTITY": ACT_NONE, "CUDNN_ACTIVATION_SIGMOID": ACT_SIGMOID, "CUDNN_ACTIVATION_TANH": ACT_TANH}


def _pointer(t):
    return t.Pointer if t is not None else None


class BlockNorm:
    """The join between two blocks: kinds of the two norms ("rms", "layer" or None), the factor of the block's output and
    the activation of its gate.  Tensors of the stream (x, u and their gradients) have one type, those of the blocks (y, h, a
    gate in rows and their gradients) another or the same; weights, biases and a gate vector are float32."""

    def __init__(self, embeddingDim, preNorm="rms", postNorm=None, residualScale=1.0, gateActivation=None, epsilon=1e-5, gpu_wrapper=None):
        if preNorm not in _NORMS or postNorm not in _NORMS:
            raise ValueError("norms are 'rms', 'layer' or None, not %r and %r" % (preNorm, postNorm))
        if gateActivation not in _GATES:
            raise SharpNetHipError(CublasStatus.CUBLAS_STATUS_NOT_SUPPORTED, "gate activation %r" % (gateActivation,))
        self.EmbeddingDim = int(embeddingDim)
        self.PreNorm, self.PostNorm, self.GateActivation = _NORMS[preNorm], _NORMS[postNorm], _GATES[gateActivation]
        self.ResidualScale, self.Epsilon = float(residualScale), float(epsilon)
        self.Wrapper = gpu_wrapper
        self._workspace = None
        self._workspaceBytes = 0

    def _rows(self, t, name, rows, type_=None):
        if t is None:
            return
        t.AssertIsNotDisposed()
        if t.Shape[-1] != self.EmbeddingDim or t.Count != rows * self.EmbeddingDim:
            raise ValueError("%s is %s, expected %d rows of %d" % (name, t.Shape, rows, self.EmbeddingDim))
        if type_ is not None and t.Type != type_:
            raise ValueError("%s is %s, expected %s" % (name, t.Type, type_))

    def _vector(self, t, name):
        if t is None:
            return
        t.AssertIsNotDisposed()
        if t.Count != self.EmbeddingDim or t.Type != "float32":
            raise ValueError("%s is %s %s, expected %d float32" % (name, t.Type, t.Shape, self.EmbeddingDim))

    def _desc(self, stream, blocks, rows, y, gate, gateRows, preWeight, preBias, postWeight, postBias, preStatistics, postStatistics):
        block = next((t for t in blocks if t is not None), stream)
        for t in blocks:
            self._rows(t, "a tensor of the blocks", rows, block.Type)
        for t, name in ((preWeight, "preWeight"), (preBias, "preBias"), (postWeight, "postWeight"), (postBias, "postBias")):
            self._vector(t, name)
        for t, name in ((preStatistics, "preStatistics"), (postStatistics, "postStatistics")):
            if t is not None and (t.Count != 2 * rows or t.Type != "float32"):
                raise ValueError("%s is %s %s, expected (%d, 2) float32" % (name, t.Type, t.Shape, rows))
        if gate is not None and gateRows == 0:
            self._vector(gate, "gate")
        elif gate is not None:
            if gateRows < 0:
                raise ValueError("gateRows is %d" % gateRows)
            self._rows(gate, "gate", -(-rows // gateRows), block.Type)
        for t in (stream, block):
            if t.Type not in ("float32", "bfloat16"):
                raise ValueError("rows must be float32 or bfloat16, not %s" % t.Type)
        return BlockNormDesc(stream_type=TYPES[stream.Type], block_type=TYPES[block.Type], pre_norm=self.PreNorm, post_norm=self.PostNorm,
                             gate_activation=self.GateActivation, dim=self.EmbeddingDim, gate_rows=gateRows, rows=rows,
                             epsilon=self.Epsilon, residual_scale=self.ResidualScale, pre_weight=_pointer(preWeight),
                             pre_bias=_pointer(preBias), post_weight=_pointer(postWeight), post_bias=_pointer(postBias),
                             gate=_pointer(gate), y=_pointer(y), pre_statistics=_pointer(preStatistics),
                             post_statistics=_pointer(postStatistics))

    def _row_count(self, t):
        if self.EmbeddingDim <= 0 or t.Shape[-1] != self.EmbeddingDim:
            raise ValueError("rows of %s do not fit an embedding dimension of %d" % (t.Shape, self.EmbeddingDim))
        return t.Count // self.EmbeddingDim

    def ForwardPropagation(self, x, h, y=None, u=None, gate=None, gateRows=0, preWeight=None, preBias=None, postWeight=None,
                           postBias=None, preStatistics=None, postStatistics=None):
        """h and u from x and y; h is None for a join without a norm ahead of the next block, y and u for a norm without a
        block.  gateRows: rows that share a row of the gate (0: the gate is one vector)."""
        rows = self._row_count(x)
        d = self._desc(x, (y, h), rows, y, gate, gateRows, preWeight, preBias, postWeight, postBias, preStatistics, postStatistics)
        self._rows(x, "x", rows)
        self._rows(u, "u", rows, x.Type)
        d.x, d.u, d.h = x.Pointer, _pointer(u), _pointer(h)
        check_status(x._lib.snhip_block_norm_forward(x.Wrapper.handle, ctypes.byref(d)), "snhip_block_norm_forward")

    def BackwardPropagation(self, dx, u, dh, du=None, y=None, dy=None, gate=None, dGate=None, gateRows=0, preWeight=None,
                            preStatistics=None, dPreWeight=None, dPreBias=None, postWeight=None, postBias=None, postStatistics=None,
                            dPostWeight=None, dPostBias=None, accumulate=False, workspace=None):
        """dx and dy from dh and du (either may be None), with the forward pass's u, y, gate and statistics; gradients that are
        None are skipped, ``accumulate`` adds to those of the vectors.  Without a ``workspace`` the layer keeps one of its
        own (see WordEmbedding.BackwardPropagation)."""
        rows = self._row_count(dx)
        d = self._desc(dx, (y, dh, dy), rows, y, gate, gateRows, preWeight, None, postWeight, postBias, preStatistics, postStatistics)
        for t, name in ((dx, "dx"), (u, "u"), (du, "du")):
            self._rows(t, name, rows, dx.Type)
        for t, name in ((dPreWeight, "dPreWeight"), (dPreBias, "dPreBias"), (dPostWeight, "dPostWeight"), (dPostBias, "dPostBias")):
            self._vector(t, name)
        if dGate is not None and (gate is None or dGate.Shape != gate.Shape or dGate.Type != gate.Type):
            raise ValueError("dGate must have the gate's shape and type")
        d.u, d.dx, d.dh, d.du, d.dy = _pointer(u), dx.Pointer, _pointer(dh), _pointer(du), _pointer(dy)
        d.d_gate, d.d_pre_weight, d.d_pre_bias = _pointer(dGate), _pointer(dPreWeight), _pointer(dPreBias)
        d.d_post_weight, d.d_post_bias, d.accumulate = _pointer(dPostWeight), _pointer(dPostBias), int(bool(accumulate))
        need = ctypes.c_size_t()
        check_status(dx._lib.snhip_block_norm_backward_workspace_size(ctypes.byref(d), ctypes.byref(need)),
                     "snhip_block_norm_backward_workspace_size")
        if workspace is None and need.value:
            if self._workspaceBytes < need.value:
                if self._workspace is not None:
                    self._workspace.Wrapper.synchronize()
                    self._workspace.Dispose()
                self._workspace = GPUTensor([need.value], None, dx.Wrapper, element_type="uint8")
                self._workspaceBytes = need.value
            workspace = self._workspace
        nbytes = workspace.Count * workspace.ElementBytes if workspace is not None else 0
        check_status(dx._lib.snhip_block_norm_backward(dx.Wrapper.handle, ctypes.byref(d), _pointer(workspace), nbytes),
                     "snhip_block_norm_backward")

    def Dispose(self):
        if self._workspace is not None:
            self._workspace.Dispose()
        self._workspace, self._workspaceBytes = None, 0
