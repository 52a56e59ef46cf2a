"""Host side of the norms before and after a block (the layer and RMS norms of Prod/GPU/Kernels/SinglePrecision.cu:32-284
fused with the residual connection around a block) on GPUTensor.

``u = x + residualScale * act(gate) * N_post(y)`` and ``h = N_pre(u)``, forward and backward, each in one pass over the rows
in libsharpnet_hip.so.  x is the residual stream, y the output of the block behind it (MultiheadAttention, Linear ...), h
what the next block reads.
"""
import ctypes
import math
import threading

from .gpu_tensor import LayerWorkspace, pointer_on, stream_of
from .hiplib import (ACT_NONE, ACT_SIGMOID, ACT_TANH, BlockNormDesc, NORM_LAYER, NORM_NONE, NORM_RMS, SharpNetHipError, CublasStatus,
                     TYPES, check_status)

_NORMS = {None: NORM_NONE, "none": NORM_NONE, "rms": NORM_RMS, "layer": NORM_LAYER}
_GATES = {None: ACT_NONE, "none": ACT_NONE, "sigmoid": ACT_SIGMOID, "tanh": ACT_TANH,
          "CUDNN_ACTIVATION_IDENTITY": ACT_NONE, "CUDNN_ACTIVATION_SIGMOID": ACT_SIGMOID, "CUDNN_ACTIVATION_TANH": ACT_TANH}
_ROW_TYPES = {k: TYPES[k] for k in ("float32", "bfloat16")}


class BlockNorm:
    """The join between two blocks: kinds of the two norms ("rms", "layer" or None), the factor of the block's output and
    the activation of its gate.  Tensors of the stream (x, u and their gradients) have one type, those of the blocks (y, h, a
    gate in rows and their gradients) another or the same; weights, biases and a gate vector are float32.  Calls go to gpu_wrapper,
    without one to the wrapper of the stream's tensors."""

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

    def __setattr__(self, name, value):
        object.__setattr__(self, name, value)
        if name in ("EmbeddingDim", "PreNorm", "PostNorm", "GateActivation"):
            object.__setattr__(self, "_kind", object())  # what a thread has laid out for calls of the layer as it was is over

    def _rows(self, w, t, name, shape, type_):
        """The address of t, which is None or has rows like those of shape, in the given type, on the wrapper's device."""
        if t is None:
            return None
        if t.Shape != shape and (t.Shape[-1] != self.EmbeddingDim or math.prod(t.Shape) != math.prod(shape)):
            raise ValueError("%s is %s, expected the rows of %s" % (name, t.Shape, shape))
        if t.Type != type_:
            raise ValueError("%s is %s, expected %s" % (name, t.Type, type_))
        return pointer_on(w, t)

    def _vector(self, w, t, name):
        if t is None:
            return None
        if t.Type != "float32" or (t.Shape != self._vectorShape and math.prod(t.Shape) != self.EmbeddingDim):
            raise ValueError("%s is %s %s, expected %d float32" % (name, t.Type, t.Shape, self.EmbeddingDim))
        return pointer_on(w, t)

    def _statistics(self, w, t, name, rows):
        if t is None:
            return None
        if t.Type != "float32" or math.prod(t.Shape) != 2 * rows:
            raise ValueError("%s is %s %s, expected (%d, 2) float32" % (name, t.Type, t.Shape, rows))
        return pointer_on(w, t)

    def _desc(self, direction, stream, block, gate, gateRows, preWeight, preBias, postWeight, postBias, preStatistics, postStatistics):
        """What both directions have: the layer itself, sizes and types, gate, weights, statistics."""
        w, dim, stream_type, block_type = self.Wrapper or stream.Wrapper, self.EmbeddingDim, stream.Type, block.Type
        if dim <= 0 or stream.Shape[-1] != dim:
            raise ValueError("rows of %s do not fit an embedding dimension of %d" % (stream.Shape, dim))
        if stream_type not in _ROW_TYPES or block_type not in _ROW_TYPES:
            raise ValueError("rows must be float32 or bfloat16, not %s and %s" % (stream_type, block_type))
        if gateRows < 0:
            raise ValueError("gateRows is %d" % gateRows)
        rows, mine = math.prod(stream.Shape) // dim, self._mine.__dict__
        if mine.get("kind") is not self._kind:  # (the first call, or the layer has been changed)
            mine.clear()
            mine["kind"], self._vectorShape = self._kind, [dim]
        d = mine.get(direction)
        if d is None:
            d = mine[direction] = BlockNormDesc(pre_norm=self.PreNorm, post_norm=self.PostNorm, gate_activation=self.GateActivation, dim=dim)
        d.epsilon, d.residual_scale = self.Epsilon, self.ResidualScale
        d.rows, d.gate_rows = rows, min(gateRows, 0x7FFFFFFF)  # (there are no more rows)
        d.stream_type, d.block_type = _ROW_TYPES[stream_type], _ROW_TYPES[block_type]
        d.pre_weight, d.pre_bias = self._vector(w, preWeight, "preWeight"), self._vector(w, preBias, "preBias")
        d.post_weight, d.post_bias = self._vector(w, postWeight, "postWeight"), self._vector(w, postBias, "postBias")
        d.pre_statistics = self._statistics(w, preStatistics, "preStatistics", rows)
        d.post_statistics = self._statistics(w, postStatistics, "postStatistics", rows)
        if gateRows == 0:
            d.gate = self._vector(w, gate, "gate")
        else:
            d.gate = self._rows(w, gate, "gate", [-(-rows // gateRows), dim], block_type)
        return d

    def ForwardPropagation(self, x, h, y=None, u=None, gate=None, gateRows=0, preWeight=None, preBias=None, postWeight=None,
                           postBias=None, preStatistics=None, postStatistics=None):
        """h and u from x and y; h is None for a join without a norm ahead of the next block, y and u for a norm without a
        block.  gateRows: rows that share a row of the gate (0: the gate is one vector)."""
        shape, w, stream_type = x.Shape, self.Wrapper or x.Wrapper, x.Type
        block = h if h is not None else y if y is not None else x
        block_type = block.Type
        if (y is None and u is not None) or (not self.PreNorm and (h is not None or preStatistics is not None)) or \
                (postStatistics is not None and not self.PostNorm):
            raise ValueError("there is no u without y, and neither h nor statistics without their norm")
        d = self._desc("forward", x, block, gate, gateRows, preWeight, preBias, postWeight, postBias, preStatistics, postStatistics)
        d.x, d.u = pointer_on(w, x), self._rows(w, u, "u", shape, stream_type)
        d.y, d.h = self._rows(w, y, "y", shape, block_type), self._rows(w, h, "h", shape, block_type)
        check_status(x._lib.snhip_block_norm_forward(w.handle, ctypes.byref(d)), "snhip_block_norm_forward")

    def BackwardPropagation(self, dx, u, dh, du=None, y=None, dy=None, gate=None, dGate=None, gateRows=0, preWeight=None,
                            preStatistics=None, dPreWeight=None, dPreBias=None, postWeight=None, postBias=None, postStatistics=None,
                            dPostWeight=None, dPostBias=None, accumulate=False, workspace=None):
        """dx and dy from dh and du (either may be None), with the forward pass's u, y, gate and statistics (y also where its values
        do not matter: without it there is no block and no dy); gradients that are None are skipped, ``accumulate`` adds to those of
        the vectors.  Without a ``workspace`` the layer keeps one of its
        own (see WordEmbedding.BackwardPropagation)."""
        shape, w, lib, stream_type = dx.Shape, self.Wrapper or dx.Wrapper, dx._lib, dx.Type
        block = dh if dh is not None else y if y is not None else dy if dy is not None else dx
        block_type = block.Type
        if dy is not None and y is None:
            raise ValueError("dy is wanted without y")
        d = self._desc("backward", dx, block, gate, gateRows, preWeight, None, postWeight, postBias, preStatistics, postStatistics)
        d.dx, d.u, d.du = pointer_on(w, dx), self._rows(w, u, "u", shape, stream_type), self._rows(w, du, "du", shape, stream_type)
        d.dh, d.y = self._rows(w, dh, "dh", shape, block_type), self._rows(w, y, "y", shape, block_type)
        d.dy = self._rows(w, dy, "dy", shape, block_type)
        if dGate is not None and (gate is None or dGate.Shape != gate.Shape or dGate.Type != gate.Type):
            raise ValueError("dGate must have the gate's shape and type")
        d.d_gate = pointer_on(w, dGate)
        d.d_pre_weight, d.d_pre_bias = self._vector(w, dPreWeight, "dPreWeight"), self._vector(w, dPreBias, "dPreBias")
        d.d_post_weight, d.d_post_bias = self._vector(w, dPostWeight, "dPostWeight"), self._vector(w, dPostBias, "dPostBias")
        d.accumulate = 1 if accumulate else 0
        if workspace is None:
            # what its size depends on
            call = (shape, stream_type, block_type, gateRows, dh is None, gate is None, dGate is None, dPreWeight is None,
                    dPreBias is None, dPostWeight is None, dPostBias is None)
            mine = self._mine.__dict__
            if mine.get("call") != call:
                need = ctypes.c_size_t()
                check_status(lib.snhip_block_norm_backward_workspace_size(ctypes.byref(d), ctypes.byref(need)),
                             "snhip_block_norm_backward_workspace_size")
                mine["call"], mine["need"] = (list(shape),) + call[1:], need.value
            workspace = self._workspace.Get(w, mine["need"], stream_of(w)) if mine["need"] > 0 else None
            nbytes = workspace.Shape[0] if workspace is not None else 0
        else:
            nbytes = workspace.Count * workspace.ElementBytes
        check_status(lib.snhip_block_norm_backward(w.handle, ctypes.byref(d), pointer_on(w, workspace), nbytes),
                     "snhip_block_norm_backward")

    def Dispose(self):
        self._workspace.Dispose()
