"""Host side of the word embedding (WordEmbeddingForwardPropagation / WordEmbeddingBackwardPropagation,
Prod/GPU/Kernels/SinglePrecision.cu:617,650) on GPUTensor.

``y[t] = scale * W[x[t]]`` for every token t and the gradient of W, both in libsharpnet_hip.so.  The ids in ``x`` may be
float32 (the reference's form, rounded toward zero), int32 or int64; an id outside [0, vocabularySize) is no token: its
row of y is zeros and it adds nothing to the gradient.
"""
import ctypes
import math

from .gpu_tensor import GPUTensor
from .hiplib import EmbeddingDesc, TYPES, check_status

_ID_TYPES = {k: TYPES[k] for k in ("float32", "int32", "int64")}
_ROW_TYPES = {k: TYPES[k] for k in ("float32", "bfloat16")}


class WordEmbedding:
    """The layer: sizes, scale and the scratch memory of its backward pass."""

    def __init__(self, vocabularySize, embeddingDim, scale=1.0, paddingIndex=-1, gpu_wrapper=None):
        if vocabularySize < 0 or embeddingDim < 0 or paddingIndex < -1:
            raise ValueError("vocabularySize %d, embeddingDim %d, paddingIndex %d" % (vocabularySize, embeddingDim, paddingIndex))
        self.VocabularySize, self.EmbeddingDim = int(vocabularySize), int(embeddingDim)
        self.Scale, self.PaddingIndex = float(scale), int(paddingIndex)
        self.Wrapper = gpu_wrapper
        self._workspace = None
        self._workspaceBytes = 0
        # a call fills in every field that is not of the layer itself
        self._d = EmbeddingDesc(vocabulary=self.VocabularySize, dim=self.EmbeddingDim, padding_index=self.PaddingIndex, scale=self.Scale)
        self._need = ctypes.c_size_t()

    def _desc(self, x, rows, table_type):
        """rows: y or dy, (..., EmbeddingDim) with one row per id of x."""
        if x.Type not in _ID_TYPES:
            raise ValueError("ids must be float32, int32 or int64, not %s" % x.Type)
        if rows.Type not in _ROW_TYPES or table_type not in _ROW_TYPES:
            raise ValueError("rows and table must be float32 or bfloat16, not %s and %s" % (rows.Type, table_type))
        tokens = math.prod(x.Shape)
        if rows.Shape[-1] != self.EmbeddingDim or math.prod(rows.Shape) != tokens * self.EmbeddingDim:
            raise ValueError("%s ids and rows of %s do not fit an embedding dimension of %d" % (x.Shape, rows.Shape, self.EmbeddingDim))
        d = self._d
        d.id_type, d.table_type, d.output_type, d.tokens = _ID_TYPES[x.Type], _ROW_TYPES[table_type], _ROW_TYPES[rows.Type], tokens
        return d

    def _check_table(self, table):
        if table.Shape != [self.VocabularySize, self.EmbeddingDim]:
            raise ValueError("the table must be %s, not %s" % ([self.VocabularySize, self.EmbeddingDim], table.Shape))

    def ForwardPropagation(self, y, x, wordEmbedding):
        """y (ids' shape + EmbeddingDim) = Scale * wordEmbedding[x]."""
        self._check_table(wordEmbedding)
        d = self._desc(x, y, wordEmbedding.Type)
        y.AssertIsNotDisposed()
        x.AssertIsNotDisposed()
        wordEmbedding.AssertIsNotDisposed()
        check_status(y._lib.snhip_embedding_forward(y.Wrapper.handle, ctypes.byref(d), x.Pointer, wordEmbedding.Pointer,
                                                    y.Pointer), "snhip_embedding_forward")

    def BackwardWorkspaceSize(self, x, dy):
        nbytes = ctypes.c_size_t()
        d = self._desc(x, dy, "float32")
        check_status(dy._lib.snhip_embedding_backward_workspace_size(ctypes.byref(d), ctypes.byref(nbytes)),
                     "snhip_embedding_backward_workspace_size")
        return nbytes.value

    def BackwardPropagation(self, dWordEmbedding, x, dy, accumulate=False, workspace=None):
        """dWordEmbedding (float32) = the table's gradient, or += it with ``accumulate``.  Without a ``workspace`` the layer
        keeps one of its own, which grows when a longer batch comes (an allocation: size it with a first call before a
        stream capture) and belongs to one stream at a time."""
        self._check_table(dWordEmbedding)
        if dWordEmbedding.Type != "float32":
            raise ValueError("the table's gradient must be float32, not %s" % dWordEmbedding.Type)
        d = self._desc(x, dy, "float32")
        dWordEmbedding.AssertIsNotDisposed()
        x.AssertIsNotDisposed()
        dy.AssertIsNotDisposed()
        need = self._need
        check_status(dy._lib.snhip_embedding_backward_workspace_size(ctypes.byref(d), ctypes.byref(need)),
                     "snhip_embedding_backward_workspace_size")
        if workspace is None and need.value:
            if self._workspaceBytes < need.value:
                if self._workspace is not None:
                    self._workspace.Wrapper.synchronize()
                    self._workspace.Dispose()
                self._workspace = GPUTensor([need.value], None, dy.Wrapper, element_type="uint8")
                self._workspaceBytes = need.value
            workspace = self._workspace
        check_status(dy._lib.snhip_embedding_backward(dy.Wrapper.handle, ctypes.byref(d), x.Pointer, dy.Pointer,
                                                      dWordEmbedding.Pointer, int(bool(accumulate)),
                                                      workspace.Pointer if workspace is not None else None,
                                                      workspace.Count * workspace.ElementBytes if workspace is not None else 0),
                     "snhip_embedding_backward")

    def Dispose(self):
        if self._workspace is not None:
            self._workspace.Dispose()
        self._workspace, self._workspaceBytes = None, 0
