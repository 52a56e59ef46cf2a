"""Host side of the word embedding (WordEmbeddingForwardPropagation / WordEmbeddingBackwardPropagation,
Prod/GPU/Kernels/SinglePrecision.cu:617,650) on GPUTensor.

``y[t] = scale * W[x[t]]`` for every token t and the gradient of W, both in libsharpnet_hip.so.  The ids in ``x`` may be
float32 (the reference's form, rounded toward zero), int32 or int64; an id outside [0, vocabularySize) is no token: its
row of y is zeros and it adds nothing to the gradient.
"""
import ctypes
import math
import threading

from .gpu_tensor import LayerWorkspace, pointer_on, stream_of
from .hiplib import EmbeddingDesc, TYPES, check_status

_ID_TYPES = {k: TYPES[k] for k in ("float32", "int32", "int64")}
_ROW_TYPES = {k: TYPES[k] for k in ("float32", "bfloat16")}


class WordEmbedding:
    """The layer: sizes, scale and the scratch memory of its backward pass.  Its calls go to gpu_wrapper, without one to the wrapper
    of the rows they are given."""

    def __init__(self, vocabularySize, embeddingDim, scale=1.0, paddingIndex=-1, gpu_wrapper=None):
        if vocabularySize < 0 or embeddingDim < 0 or paddingIndex < -1:
            raise ValueError("vocabularySize %d, embeddingDim %d, paddingIndex %d" % (vocabularySize, embeddingDim, paddingIndex))
        self.VocabularySize, self.EmbeddingDim = int(vocabularySize), int(embeddingDim)
        self.Scale, self.PaddingIndex = float(scale), int(paddingIndex)
        self.Wrapper = gpu_wrapper
        self._workspace = LayerWorkspace()
        self._mine = threading.local()  # for each thread: its last call's sizes and types, and their descriptor

    def _desc(self, x, rows, table_type):
        """rows: y or dy, (..., EmbeddingDim) with one row per id of x."""
        tokens, mine, dim = math.prod(x.Shape), self._mine.__dict__, self.EmbeddingDim
        if rows.Shape[-1] != dim or math.prod(rows.Shape) != tokens * dim:
            raise ValueError("%s ids and rows of %s do not fit an embedding dimension of %d" % (x.Shape, rows.Shape, dim))
        call = (x.Type, table_type, rows.Type, tokens, self.VocabularySize, dim, self.PaddingIndex, self.Scale)
        if mine.get("call") != call:
            if x.Type not in _ID_TYPES:
                raise ValueError("ids must be float32, int32 or int64, not %s" % x.Type)
            if rows.Type not in _ROW_TYPES or table_type not in _ROW_TYPES:
                raise ValueError("rows and table must be float32 or bfloat16, not %s and %s" % (rows.Type, table_type))
            mine["desc"] = EmbeddingDesc(id_type=_ID_TYPES[x.Type], table_type=_ROW_TYPES[table_type], output_type=_ROW_TYPES[rows.Type],
                                         tokens=tokens, vocabulary=self.VocabularySize, dim=dim, scale=self.Scale,
                                         padding_index=self.PaddingIndex if self.PaddingIndex < self.VocabularySize else -1)
            mine["call"], mine["need"] = call, None
        return mine["desc"]

    def _check_table(self, table):
        if table.Shape != [self.VocabularySize, self.EmbeddingDim]:
            raise ValueError("the table must be %s, not %s" % ([self.VocabularySize, self.EmbeddingDim], table.Shape))

    def ForwardPropagation(self, y, x, wordEmbedding):
        """y (ids' shape + EmbeddingDim) = Scale * wordEmbedding[x]."""
        self._check_table(wordEmbedding)
        d, w = self._desc(x, y, wordEmbedding.Type), self.Wrapper or y.Wrapper
        check_status(y._lib.snhip_embedding_forward(w.handle, ctypes.byref(d), pointer_on(w, x), pointer_on(w, wordEmbedding),
                                                    pointer_on(w, y)), "snhip_embedding_forward")

    def BackwardWorkspaceSize(self, x, dy):
        nbytes = ctypes.c_size_t()
        d = self._desc(x, dy, "float32")
        check_status(dy._lib.snhip_embedding_backward_workspace_size(ctypes.byref(d), ctypes.byref(nbytes)),
                     "snhip_embedding_backward_workspace_size")
        return nbytes.value

    def BackwardPropagation(self, dWordEmbedding, x, dy, accumulate=False, workspace=None):
        """dWordEmbedding (float32) = the table's gradient, or += it with ``accumulate``.  Without a ``workspace`` the layer
        keeps one of its own for each wrapper and stream that it is called on, which grows when a longer batch comes.  It is one
        call's at a time: graphs whose replays may overlap one another, or calls on the stream they were captured on, get one each."""
        self._check_table(dWordEmbedding)
        if dWordEmbedding.Type != "float32":
            raise ValueError("the table's gradient must be float32, not %s" % dWordEmbedding.Type)
        d, w, mine = self._desc(x, dy, "float32"), self.Wrapper or dy.Wrapper, self._mine.__dict__
        pointers = pointer_on(w, x), pointer_on(w, dy), pointer_on(w, dWordEmbedding)
        if workspace is None:
            if mine["need"] is None:
                mine["need"] = self.BackwardWorkspaceSize(x, dy)
            workspace = self._workspace.Get(w, mine["need"], stream_of(w)) if mine["need"] > 0 else None
        check_status(dy._lib.snhip_embedding_backward(w.handle, ctypes.byref(d), *pointers, int(bool(accumulate)),
                                                      pointer_on(w, workspace),
                                                      workspace.Count * workspace.ElementBytes if workspace is not None else 0),
                     "snhip_embedding_backward")

    def Dispose(self):
        self._workspace.Dispose()
