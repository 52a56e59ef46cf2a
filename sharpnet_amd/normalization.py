"""Host side of the norms before and after a block (the layer and RMS norms of Prod/GPU/Kernels/SinglePrecision.cu:32-284
fused with the residual connection around a block) on GPUTensor.

``u = x + residualScale * act(gate) * N_post(y)`` and ``h = N_pre(u)``, forward and backward, each in one pass over the rows
in libsharpnet_hip.so.  x is the residual stream, y the output of the block behind it (MultiheadAttention, Linear ...), h
what the next block reads.
"""
import ctypes
import math
import threading

from .gpu_tensor import LayerWorkspace, pointer_on
from .hiplib import (ACT_NONE, ACT_SIGMOID, ACT_TANH, BlockNormDesc, NORM_LAYER, NORM_NONE, NORM_RMS, SharpNetHipError, CublasStatus,
                     TYPES, check_status)

_NORMS = {None: NORM_NONE, "none": NORM_NONE, "rms": NORM_RMS, "layer": NORM_LAYER}
_GATES = {None: ACT_NONE, "none": ACT_NONE, "sigmoid": ACT_SIGMOID, "tanh": ACT_TANH,
          "CUDNN_ACTIVATION_IDENTITY": ACT_NONE, "CUDNN_ACTIVATION_SIGMOID": ACT_SIGMOID, "CUDNN_ACTIVATION_TANH": ACT_TANH}
_ROW_TYPES = {k: TYPES[k] for k in ("float32", "bfloat16")}


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
        self._vectorShape = [self.EmbeddingDim]
        self.PreNorm, self.PostNorm, self.GateActivation = _NORMS[preNorm], _NORMS[postNorm], _GATES[gateActivation]
        self.ResidualScale, self.Epsilon = float(residualScale), float(epsilon)
        self.Wrapper = gpu_wrapper
        self._workspace = LayerWorkspace()
        self._mine = threading.local()  # a descriptor for each thread and direction; a call fills in what is not the layer's kind

    def _rows(self, t, name, shape, type_):
        """t is None or has rows like those of shape, in the given type."""
        if t is None:
            return
        if t.Shape != shape and (t.Shape[-1] != self.EmbeddingDim or math.prod(t.Shape) != math.prod(shape)):
            raise ValueError("%s is %s, expected the rows of %s" % (name, t.Shape, shape))
        if t.Type != type_:
            raise ValueError("%s is %s, expected %s" % (name, t.Type, type_))

    def _vector(self, t, name):
        if t is not None and (t.Type != "float32" or (t.Shape != self._vectorShape and math.prod(t.Shape) != self.EmbeddingDim)):
            raise ValueError("%s is %s %s, expected %d float32" % (name, t.Type, t.Shape, self.EmbeddingDim))

    def _desc(self, direction, stream, block, gate, gateRows, preWeight, preBias, postWeight, postBias, preStatistics, postStatistics):
        """What both directions have: the layer itself, sizes and types, gate, weights, statistics."""
        if self.EmbeddingDim <= 0 or stream.Shape[-1] != self.EmbeddingDim:
            raise ValueError("rows of %s do not fit an embedding dimension of %d" % (stream.Shape, self.EmbeddingDim))
        if stream.Type not in _ROW_TYPES or block.Type not in _ROW_TYPES:
            raise ValueError("rows must be float32 or bfloat16, not %s and %s" % (stream.Type, block.Type))
        rows = math.prod(stream.Shape) // self.EmbeddingDim
        self._vector(preWeight, "preWeight")
        self._vector(preBias, "preBias")
        self._vector(postWeight, "postWeight")
        self._vector(postBias, "postBias")
        for t, name in ((preStatistics, "preStatistics"), (postStatistics, "postStatistics")):
            if t is not None and (math.prod(t.Shape) != 2 * rows or t.Type != "float32"):
                raise ValueError("%s is %s %s, expected (%d, 2) float32" % (name, t.Type, t.Shape, rows))
        if gateRows < 0:
            raise ValueError("gateRows is %d" % gateRows)
        if gate is not None:
            if gateRows == 0:
                self._vector(gate, "gate")
            else:
                self._rows(gate, "gate", [-(-rows // gateRows), self.EmbeddingDim], block.Type)
        w, mine = stream.Wrapper, self._mine.__dict__
        d = mine.get(direction)
        if d is None:
            d = mine[direction] = BlockNormDesc(pre_norm=self.PreNorm, post_norm=self.PostNorm, gate_activation=self.GateActivation,
                                                dim=self.EmbeddingDim)
        d.epsilon, d.residual_scale = self.Epsilon, self.ResidualScale
        d.rows, d.gate_rows = rows, gateRows
        d.stream_type, d.block_type = _ROW_TYPES[stream.Type], _ROW_TYPES[block.Type]
        d.gate, d.pre_weight, d.pre_bias = pointer_on(w, gate), pointer_on(w, preWeight), pointer_on(w, preBias)
        d.post_weight, d.post_bias = pointer_on(w, postWeight), pointer_on(w, postBias)
        d.pre_statistics, d.post_statistics = pointer_on(w, preStatistics), pointer_on(w, postStatistics)
        return d

    def ForwardPropagation(self, x, h, y=None, u=None, gate=None, gateRows=0, preWeight=None, preBias=None, postWeight=None,
                           postBias=None, preStatistics=None, postStatistics=None):
        """h and u from x and y; h is None for a join without a norm ahead of the next block, y and u for a norm without a
        block.  gateRows: rows that share a row of the gate (0: the gate is one vector)."""
        shape, w = x.Shape, x.Wrapper
        block = h if h is not None else y if y is not None else x
        d = self._desc("forward", x, block, gate, gateRows, preWeight, preBias, postWeight, postBias, preStatistics, postStatistics)
        self._rows(y, "y", shape, block.Type)
        self._rows(h, "h", shape, block.Type)
        self._rows(u, "u", shape, x.Type)
        d.x, d.y, d.u, d.h = pointer_on(w, x), pointer_on(w, y), pointer_on(w, u), pointer_on(w, h)
        check_status(x._lib.snhip_block_norm_forward(w.handle, ctypes.byref(d)), "snhip_block_norm_forward")

    def BackwardPropagation(self, dx, u, dh, du=None, y=None, dy=None, gate=None, dGate=None, gateRows=0, preWeight=None,
                            preStatistics=None, dPreWeight=None, dPreBias=None, postWeight=None, postBias=None, postStatistics=None,
                            dPostWeight=None, dPostBias=None, accumulate=False, workspace=None):
        """dx and dy from dh and du (either may be None), with the forward pass's u, y, gate and statistics; gradients that are
        None are skipped, ``accumulate`` adds to those of the vectors.  Without a ``workspace`` the layer keeps one of its
        own (see WordEmbedding.BackwardPropagation)."""
        shape, w = dx.Shape, dx.Wrapper
        block = next((t for t in (dh, y, dy) if t is not None), dx)
        d = self._desc("backward", dx, block, gate, gateRows, preWeight, None, postWeight, postBias, preStatistics, postStatistics)
        for t, name in ((y, "y"), (dh, "dh"), (dy, "dy")):
            self._rows(t, name, shape, block.Type)
        for t, name in ((u, "u"), (du, "du")):
            self._rows(t, name, shape, dx.Type)
        for t, name in ((dPreWeight, "dPreWeight"), (dPreBias, "dPreBias"), (dPostWeight, "dPostWeight"), (dPostBias, "dPostBias")):
            self._vector(t, name)
        if dGate is not None and (gate is None or dGate.Shape != gate.Shape or dGate.Type != gate.Type):
            raise ValueError("dGate must have the gate's shape and type")
        d.y, d.u, d.dx, d.dh, d.du, d.dy = (pointer_on(w, t) for t in (y, u, dx, dh, du, dy))
        d.d_gate, d.d_pre_weight, d.d_pre_bias = pointer_on(w, dGate), pointer_on(w, dPreWeight), pointer_on(w, dPreBias)
        d.d_post_weight, d.d_post_bias = pointer_on(w, dPostWeight), pointer_on(w, dPostBias)
        d.accumulate = 1 if accumulate else 0
        need, lib = ctypes.c_size_t(), dx._lib
        check_status(lib.snhip_block_norm_backward_workspace_size(ctypes.byref(d), ctypes.byref(need)),
                     "snhip_block_norm_backward_workspace_size")
        if workspace is None:
            workspace = self._workspace.Get(w, need.value)
        nbytes = workspace.Count * workspace.ElementBytes if workspace is not None else 0
        check_status(lib.snhip_block_norm_backward(w.handle, ctypes.byref(d), pointer_on(w, workspace), nbytes),
                     "snhip_block_norm_backward")

    def Dispose(self):
        self._workspace.Dispose()
