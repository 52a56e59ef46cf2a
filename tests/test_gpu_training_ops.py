"""Word embedding, block norm and AdamW on the GPU against their plain 64-bit forms (training_reference.py, where the bounds
are derived)."""
import ctypes

import numpy as np
import pytest

from tests import training_reference as ref

pytestmark = pytest.mark.gpu


def tensor(w, a, type_="float32"):
    from sharpnet_amd import GPUTensor
    return GPUTensor(list(a.shape), a, w, element_type=type_)


def empty(w, shape, type_="float32"):
    """Device memory that holds NaN (or bytes of 0xff) until it is written."""
    from sharpnet_amd import GPUTensor
    t = GPUTensor(list(shape), None, w, element_type=type_)
    w.lib.snhip_memset32(w.handle, t.Pointer, 0xFFFFFFFF, t._nbytes // 4)
    return t


def within(got, want, bound, name=""):
    got = got.reshape(want.shape).astype(np.float64)
    assert np.all(np.isfinite(got)), name
    over = np.abs(got - want) - bound
    assert over.max(initial=-1.0) <= 0, "%s: %g over its bound, at %s" % (name, over.max(), np.unravel_index(over.argmax(), over.shape))


def rounded(a, type_):
    """Values that the storage type holds exactly, in float32."""
    return ref.bf16(a).astype(np.float32) if type_ == "bfloat16" else a.astype(np.float32)


# ---------------------------------------------------------------------------------------------------------------
# word embedding
# ---------------------------------------------------------------------------------------------------------------
def make_ids(rng, n, vocabulary, type_, stray=True):
    ids = np.minimum((vocabulary * rng.random(n) ** 3).astype(np.int64), vocabulary - 1)
    if stray and n >= 4:
        ids[rng.integers(0, n, n // 4)] = rng.choice([-1, -7, vocabulary, vocabulary + 5, 2 ** 31 - 1], n // 4)
    if type_ == "int64" and stray and n >= 4:
        ids[0] = 2 ** 40
    ids = ids.astype({"float32": np.float32, "int32": np.int32, "int64": np.int64}[type_])
    if type_ == "float32" and stray and n >= 8:
        ids[1], ids[3], ids[5], ids[6] = np.nan, np.inf, -np.inf, -0.25
    return ids


FORWARD = [(1, 1, 1, "int32", "float32", "float32"), (3, 7, 5, "float32", "float32", "float32"),
           (64, 1000, 1024, "int32", "bfloat16", "bfloat16"), (257, 50, 100, "int64", "float32", "bfloat16"),
           (1000, 513, 30, "float32", "bfloat16", "float32"), (5, 3, 4100, "int64", "bfloat16", "bfloat16"),
           (2049, 4000, 258, "int32", "float32", "float32")]


@pytest.mark.parametrize("tokens,vocabulary,dim,ids,table,out", FORWARD)
def test_embedding_forward(gpu_wrapper, tokens, vocabulary, dim, ids, table, out):
    from sharpnet_amd import embedding
    w, rng = gpu_wrapper, np.random.default_rng(tokens)
    x = make_ids(rng, tokens, vocabulary, ids)
    W = rounded(rng.normal(0, 1, (vocabulary, dim)), table)
    scale = 1.7
    layer = embedding.WordEmbedding(vocabulary, dim, scale)
    y = empty(w, (tokens, dim), out)
    layer.ForwardPropagation(y, tensor(w, x, ids), tensor(w, W, table))
    want = ref.embedding_forward(x, W, scale)
    got = y.ToNumpy()
    within(got, want, (ref.U + (ref.BF16 if out == "bfloat16" else 0)) * np.abs(want) * 1.001, "y")
    assert np.all(got[ref.valid_ids(x, vocabulary) < 0] == 0)


@pytest.mark.parametrize("offset,ld", [(0, 12), (1, 13), (4, 16), (2, 10)])
@pytest.mark.parametrize("out", ["float32", "bfloat16"])
def test_embedding_rows_with_pitches_and_any_alignment(gpu_wrapper, offset, ld, out):
    """Row pitches and start addresses that rule the wide accesses out (and some that do not); what lies between the rows
    stays as it was."""
    from sharpnet_amd.hiplib import EmbeddingDesc, TYPES, check_status
    w, rng = gpu_wrapper, np.random.default_rng(ld)
    tokens, vocabulary, dim = 33, 9, 10 if ld != 16 else 16
    x = make_ids(rng, tokens, vocabulary, "int32")
    W = np.full((vocabulary, ld), 7.0, np.float32)
    W[:, :dim] = rng.normal(0, 1, (vocabulary, dim))
    gW = tensor(w, np.concatenate((np.zeros(offset, np.float32), W.reshape(-1))))
    gx = tensor(w, x, "int32")
    gy = tensor(w, np.full(offset + tokens * ld, 3.0, np.float32), out)
    d = EmbeddingDesc(id_type=TYPES["int32"], output_type=TYPES[out], tokens=tokens, vocabulary=vocabulary, dim=dim, ld_table=ld,
                      ld_output=ld, scale=0.5)
    check_status(w.lib.snhip_embedding_forward(w.handle, ctypes.byref(d), gx.Pointer, gW.Pointer + 4 * offset,
                                               gy.Pointer + gy.ElementBytes * offset))
    got = gy.ToNumpy()
    assert np.all(got[:offset] == 3.0)
    got = got[offset:].reshape(tokens, ld)
    want = ref.embedding_forward(x, W[:, :dim], 0.5)
    within(got[:, :dim], want, ref.storage(out) * np.abs(want), "y")
    assert np.all(got[:, dim:] == 3.0)
    # the gradient with the same pitches
    dy = rounded(rng.normal(0, 1, (tokens, ld)), out)
    gdy = tensor(w, np.concatenate((np.zeros(offset, np.float32), dy.reshape(-1))), out)
    gdw = tensor(w, np.full(offset + vocabulary * ld, 3.0, np.float32))
    need = ctypes.c_size_t()
    check_status(w.lib.snhip_embedding_backward_workspace_size(ctypes.byref(d), ctypes.byref(need)))
    ws = empty(w, [need.value], "uint8")
    check_status(w.lib.snhip_embedding_backward(w.handle, ctypes.byref(d), gx.Pointer, gdy.Pointer + gdy.ElementBytes * offset,
                                                gdw.Pointer + 4 * offset, 0, ws.Pointer, need.value))
    got = gdw.ToNumpy()
    assert np.all(got[:offset] == 3.0)
    got = got[offset:].reshape(vocabulary, ld)
    want, bound = ref.embedding_backward(x, dy[:, :dim], vocabulary, 0.5)
    within(got[:, :dim], want, bound, "dW")
    assert np.all(got[:, dim:] == 3.0)


BACKWARD = [(1, 1, 1, "int32", "float32"), (8, 3, 4, "int64", "float32"), (9, 3, 5, "float32", "bfloat16"),
            (4000, 5003, 100, "float32", "float32"), (16389, 300, 33, "int32", "bfloat16"), (700, 140001, 8, "int64", "float32"),
            (20000, 1, 12, "int32", "float32"), (8192, 600, 4, "int32", "float32"), (8193, 600, 4, "int64", "bfloat16"),
            (9000, 140001, 8, "float32", "float32"), (4096, 256, 256, "int32", "float32"), (4097, 256, 5, "int32", "float32"),
            (1000, 131072, 9, "int64", "bfloat16"), (900, 1, 1027, "int32", "float32"), (300, 2, 1030, "int32", "bfloat16"), (70000, 7, 3, "int64", "float32"),
            (4096, 700, 256, "int64", "bfloat16"), (4096, 256, 257, "int32", "float32"), (12000, 40, 150, "int32", "float32"), (17000, 30, 700, "int64", "bfloat16")]


@pytest.mark.parametrize("tokens,vocabulary,dim,ids,rows", BACKWARD)
def test_embedding_backward(gpu_wrapper, tokens, vocabulary, dim, ids, rows):
    """Every row of the gradient, those of no token included; rows of tokens outside the vocabulary are not read (they hold
    NaN); the same bits from a second call on used scratch memory; a padding index; accumulation."""
    from sharpnet_amd import embedding
    w, rng = gpu_wrapper, np.random.default_rng(tokens)
    x = make_ids(rng, tokens, vocabulary, ids)
    dy = rounded(rng.normal(0, 1, (tokens, dim)), rows)
    gx = tensor(w, x, ids)
    t = ref.valid_ids(x, vocabulary)
    for padding in (-1, 0):
        layer = embedding.WordEmbedding(vocabulary, dim, 1.3, padding)
        read = dy.copy()
        read[(t < 0) | (t == padding)] = np.nan
        gdy, dW = tensor(w, read, rows), empty(w, (vocabulary, dim))
        layer.BackwardPropagation(dW, gx, gdy)
        want, bound = ref.embedding_backward(x, dy, vocabulary, 1.3, padding)
        got = dW.ToNumpy()
        within(got, want, bound, "dW")
        again = empty(w, (vocabulary, dim))
        layer.BackwardPropagation(again, gx, gdy)
        assert np.array_equal(got, again.ToNumpy())
        start = rng.normal(0, 1, (vocabulary, dim)).astype(np.float32)
        into = tensor(w, start)
        layer.BackwardPropagation(into, gx, gdy, accumulate=True)
        total = start.astype(np.float64) + want
        within(into.ToNumpy(), total, bound + ref.U * np.abs(total), "dW +=")
        absent = np.setdiff1d(np.arange(vocabulary), t[t != padding])
        assert np.array_equal(into.ToNumpy()[absent], start[absent])


EXACT_TOKENS = [(70000, 7, 3, "int64"), (70000, 40, 36, "int32"), (20000, 1, 12, "int32"), (40000, 30000, 20, "float32"), (9000, 140001, 8, "int32"),
                (8192, 600, 40, "int32"), (5000, 3, 300, "int64"), (4096, 1, 256, "int32"), (3000, 2000, 30, "int32"), (66000, 100, 200, "int32")]


@pytest.mark.parametrize("tokens,vocabulary,dim,ids", EXACT_TOKENS)
@pytest.mark.parametrize("rows", ["float32", "bfloat16"])
def test_embedding_gradient_loses_and_doubles_no_token(gpu_wrapper, tokens, vocabulary, dim, ids, rows):
    """Whole numbers of up to 15: every partial sum is below 2^24, so exact in whatever order, and so is the scale of 1/2: the
    gradient has the formula's bits, and one token too few or too many would show."""
    from sharpnet_amd import embedding
    w, rng = gpu_wrapper, np.random.default_rng(tokens + dim)
    x = make_ids(rng, tokens, vocabulary, ids)
    dy = (rng.integers(1, 16, (tokens, dim)) * rng.choice([-1, 1], (1, dim))).astype(np.float32)
    assert tokens * 15 < 2 ** 24
    dW = empty(w, (vocabulary, dim))
    embedding.WordEmbedding(vocabulary, dim, 0.5).BackwardPropagation(dW, tensor(w, x, ids), tensor(w, dy, rows))
    assert np.array_equal(dW.ToNumpy().reshape(vocabulary, dim), ref.embedding_backward(x, dy, vocabulary, 0.5)[0])


@pytest.mark.parametrize("tokens,words,dim", [(4000, 10, 20), (2000, 20, 256), (4096, 400, 30), (3000, 1, 129), (9000, 700, 16), (20000, 900, 40)])
def test_embedding_backward_of_ids_that_share_a_bucket(gpu_wrapper, tokens, words, dim):
    """Ids that are all multiples of 512: whatever sorts them by their low bits has them in one place."""
    from sharpnet_amd import embedding
    w, rng = gpu_wrapper, np.random.default_rng(words)
    vocabulary = 512 * words
    x = (512 * rng.integers(0, words, tokens)).astype(np.int32)
    x[: tokens // 3] = 512 * (words // 2)  # one of them is frequent
    dy = rng.normal(0, 1, (tokens, dim)).astype(np.float32)
    dW = empty(w, (vocabulary, dim))
    embedding.WordEmbedding(vocabulary, dim).BackwardPropagation(dW, tensor(w, x, "int32"), tensor(w, dy))
    within(dW.ToNumpy(), *ref.embedding_backward(x, dy, vocabulary, 1.0), "dW")


def test_embedding_without_tokens_or_columns(gpu_wrapper):
    from sharpnet_amd import embedding
    w = gpu_wrapper
    layer = embedding.WordEmbedding(5, 6)
    dW = empty(w, (5, 6))
    layer.BackwardPropagation(dW, tensor(w, np.zeros(0, np.int32), "int32"), tensor(w, np.zeros((0, 6))))
    assert np.all(dW.ToNumpy() == 0)
    layer.ForwardPropagation(tensor(w, np.zeros((0, 6))), tensor(w, np.zeros(0, np.int32), "int32"), tensor(w, np.zeros((5, 6))))
    y = empty(w, (3, 6))     # every id outside
    layer.ForwardPropagation(y, tensor(w, np.array([-1, 5, 99], np.int32), "int32"), tensor(w, np.ones((5, 6))))
    assert np.all(y.ToNumpy() == 0)


# ---------------------------------------------------------------------------------------------------------------
# block norm
# ---------------------------------------------------------------------------------------------------------------
# rows, dim, pre, post, gate rows (None: no gate, 0: a vector), activation, biases, stream, block
NORMS = [(1, 1, "layer", None, None, None, True, "float32", "float32"),
         (5, 3, "rms", "rms", 0, None, False, "float32", "float32"),
         (17, 64, "layer", "layer", 3, "sigmoid", True, "float32", "bfloat16"),
         (33, 65, "rms", None, 1, "tanh", False, "bfloat16", "bfloat16"),
         (600, 100, "layer", "rms", 7, "sigmoid", True, "float32", "float32"),
         (9, 260, "rms", "layer", 0, "sigmoid", True, "float32", "bfloat16"),
         (700, 260, "layer", "layer", 1, None, False, "float32", "float32"),
         (1030, 512, None, "rms", 0, "tanh", False, "float32", "bfloat16"),
         (3, 1001, "layer", None, None, None, True, "float32", "float32"),
         (520, 1001, "layer", "layer", 200, "sigmoid", True, "float32", "float32"),
         (600, 1024, "rms", "rms", 1, "sigmoid", False, "bfloat16", "bfloat16"),
         (7, 2048, "rms", "layer", 2, None, True, "float32", "bfloat16"),
         (530, 2044, "layer", None, 0, None, True, "float32", "float32"),
         (2, 4096, "rms", "rms", 0, None, False, "bfloat16", "bfloat16"),
         (515, 4096, "layer", "layer", 1, "tanh", True, "float32", "bfloat16"),
         (3, 8192, "layer", "rms", 2, "sigmoid", True, "float32", "float32"),
         (513, 8190, "rms", "layer", 0, None, True, "float32", "bfloat16"),
         (5000, 12, "layer", "layer", 2, "sigmoid", True, "float32", "float32"),
         (2100, 40, "rms", "rms", 1000, None, False, "float32", "float32"),
         (4100, 128, "layer", None, 0, "sigmoid", True, "bfloat16", "bfloat16"),
         (3001, 127, "layer", "rms", 5, "tanh", True, "float32", "bfloat16"), (37, 97, "rms", "layer", 0, None, False, "bfloat16", "bfloat16"),
         (4200, 700, "layer", "rms", 0, None, False, "bfloat16", "bfloat16"), (4150, 1023, "rms", "layer", 9, "sigmoid", True, "float32", "float32"),
         (600, 2600, "layer", "layer", 0, None, False, "float32", "bfloat16"), (550, 5001, "rms", None, 1, "tanh", True, "bfloat16", "bfloat16"),
         (520, 6140, "layer", "rms", None, None, False, "float32", "float32"), (6200, 1028, "rms", "layer", 0, "sigmoid", False, "float32", "bfloat16"),
         (8195, 1032, "layer", None, 4, None, True, "bfloat16", "bfloat16"),
         (900, 900, "layer", "layer", 1, "sigmoid", True, "float32", "float32"), (801, 640, "layer", "layer", 0, "tanh", True, "float32", "bfloat16"),
         (2050, 1024, "rms", "layer", 700, "tanh", True, "bfloat16", "bfloat16"), (5, 770, "rms", None, None, None, False, "float32", "bfloat16")]


def norm_case(rng, rows, dim, pre, post, gate_rows, bias, stream, block):
    c = {"x": rounded(rng.normal(0.2, 2, (rows, dim)), stream), "weights": {}}
    c["y"] = rounded(rng.normal(0.1, 1, (rows, dim)), block) if post or gate_rows is not None else None
    c["gate"] = None
    if gate_rows == 0:
        c["gate"] = rng.normal(0.5, 1, dim).astype(np.float32)
    elif gate_rows is not None:
        c["gate"] = rounded(rng.normal(0, 1, (-(-rows // gate_rows), dim)), block)
    for which, kind in (("pre", pre), ("post", post)):
        if kind:
            c["weights"][which + "_weight"] = rng.normal(1, 0.2, dim).astype(np.float32)
            if bias:
                c["weights"][which + "_bias"] = rng.normal(0, 0.2, dim).astype(np.float32)
    return c


def on_device(w, c, stream, block, gate_rows):
    g = {k: tensor(w, v) for k, v in c["weights"].items()}
    g["x"] = tensor(w, c["x"], stream)
    if c["y"] is not None:
        g["y"] = tensor(w, c["y"], block)
    if c["gate"] is not None:
        g["gate"] = tensor(w, c["gate"], "float32" if gate_rows == 0 else block)
    return g


@pytest.mark.parametrize("rows,dim,pre,post,gate_rows,activation,bias,stream,block", NORMS)
def test_block_norm_forward(gpu_wrapper, rows, dim, pre, post, gate_rows, activation, bias, stream, block):
    from sharpnet_amd import normalization
    w, rng = gpu_wrapper, np.random.default_rng(rows + dim)
    c = norm_case(rng, rows, dim, pre, post, gate_rows, bias, stream, block)
    g = on_device(w, c, stream, block, gate_rows)
    layer = normalization.BlockNorm(dim, pre, post, residualScale=0.7, gateActivation=activation, epsilon=1e-5)
    out = {"u": empty(w, (rows, dim), stream) if c["y"] is not None else None, "h": empty(w, (rows, dim), block) if pre else None,
           "pre_statistics": empty(w, (rows, 2)) if pre else None, "post_statistics": empty(w, (rows, 2)) if post else None}
    vectors = dict(preWeight=g.get("pre_weight"), preBias=g.get("pre_bias"), postWeight=g.get("post_weight"), postBias=g.get("post_bias"))
    layer.ForwardPropagation(g["x"], out["h"], y=g.get("y"), u=out["u"], gate=g.get("gate"), gateRows=gate_rows or 0,
                             preStatistics=out["pre_statistics"], postStatistics=out["post_statistics"], **vectors)
    want = ref.block_norm_forward(c["x"], c["y"], c["gate"], gate_rows or 0, pre, post, c["weights"], 0.7, 1e-5, activation, stream, block)
    assert sorted(want) == sorted(k for k, v in out.items() if v is not None)
    for name, (value, bound) in want.items():
        within(out[name].ToNumpy(), value, bound, name)
    # without statistics, u over x and h over y: the same bits
    if c["y"] is not None:
        layer.ForwardPropagation(g["x"], g["y"] if pre else None, y=g["y"], u=g["x"], gate=g.get("gate"), gateRows=gate_rows or 0, **vectors)
        assert np.array_equal(g["x"].ToNumpy(), out["u"].ToNumpy())
        if pre:
            assert np.array_equal(g["y"].ToNumpy(), out["h"].ToNumpy())


@pytest.mark.parametrize("rows,dim,pre,post,gate_rows,activation,bias,stream,block", NORMS)
def test_block_norm_backward(gpu_wrapper, rows, dim, pre, post, gate_rows, activation, bias, stream, block):
    """dx, dy and every column sum; the same bits from a second call with dx over du and dy over dh; accumulation."""
    from sharpnet_amd import normalization
    w, rng = gpu_wrapper, np.random.default_rng(rows + dim)
    c = norm_case(rng, rows, dim, pre, post, gate_rows, bias, stream, block)
    g = on_device(w, c, stream, block, gate_rows)
    du = rounded(rng.normal(0, 1, (rows, dim)), stream)
    dh = rounded(rng.normal(0, 1, (rows, dim)), block) if pre else None
    stats = {}
    if pre:
        stats["pre"] = np.concatenate(ref.statistics(c["x"], pre, 1e-5), 1).astype(np.float32)
    if post:
        stats["post"] = np.concatenate(ref.statistics(c["y"], post, 1e-5), 1).astype(np.float32)
    want = ref.block_norm_backward(c["x"], dh, du, c["y"], c["gate"], gate_rows or 0, pre, post, c["weights"], stats, 0.7, activation,
                                   stream, block)
    if not bias:
        want.pop("d_pre_bias", None), want.pop("d_post_bias", None)
    layer = normalization.BlockNorm(dim, pre, post, residualScale=0.7, gateActivation=activation)
    gdu, gdh = tensor(w, du, stream), tensor(w, dh, block) if pre else None
    gstats = {k: tensor(w, v) for k, v in stats.items()}

    def outputs():
        o = {k: empty(w, (dim,)) for k in want if k.startswith("d_")}
        o["dx"] = empty(w, (rows, dim), stream)
        o["dy"] = empty(w, (rows, dim), block) if c["y"] is not None else None
        if "d_gate" in o and gate_rows:
            o["d_gate"] = empty(w, g["gate"].Shape, block)
        return o

    def call(o, dx, dy, **kw):
        layer.BackwardPropagation(dx, g["x"], gdh, du=gdu, y=g.get("y"), dy=dy, gate=g.get("gate"), dGate=o.get("d_gate"),
                                  gateRows=gate_rows or 0, preWeight=g.get("pre_weight"), preStatistics=gstats.get("pre"),
                                  dPreWeight=o.get("d_pre_weight"), dPreBias=o.get("d_pre_bias"), postWeight=g.get("post_weight"),
                                  postBias=g.get("post_bias"), postStatistics=gstats.get("post"), dPostWeight=o.get("d_post_weight"),
                                  dPostBias=o.get("d_post_bias"), **kw)
    o = outputs()
    call(o, o["dx"], o["dy"])
    for name, (value, bound) in want.items():
        within(o[name].ToNumpy(), value, bound, name)
    first = {k: t.ToNumpy() for k, t in o.items() if t is not None}
    # in place, on the same scratch memory, the vectors' gradients added to what is there
    start = {k: rng.normal(0, 1, dim).astype(np.float32) for k in want if k.startswith("d_") and not (k == "d_gate" and gate_rows)}
    o2 = outputs()
    for k, v in start.items():
        o2[k] = tensor(w, v)
    call(o2, gdu, gdh if pre and c["y"] is not None else o2["dy"], accumulate=True)
    assert np.array_equal(gdu.ToNumpy(), first["dx"])
    if pre and c["y"] is not None:
        assert np.array_equal(gdh.ToNumpy(), first["dy"])
    for k, v in start.items():
        assert np.array_equal(o2[k].ToNumpy(), v + first[k]), k
    if gate_rows:
        assert np.array_equal(o2["d_gate"].ToNumpy(), first["d_gate"])


@pytest.mark.parametrize("activation", ["sigmoid", "tanh"])
@pytest.mark.parametrize("gate_rows", [0, 1])
def test_block_norm_gradient_of_a_saturated_gate(gpu_wrapper, activation, gate_rows):
    """The gate's gradient keeps its digits where the activation has run into its limit, the same on both sides.  With
    e = exp(-k |g|) (k = 1, 2) the slope is e / (1 + e)^2 or four times that: the exponent's product and its constant are off by
    u each, 2 u k |g| of e; the hardware's exponential and reciprocal (twice) by 2 u each, 1 + e (twice) and three products by u;
    what the slope is multiplied with by 3 u more: (16 + 2 k |g|) u."""
    from sharpnet_amd import normalization
    w, rng = gpu_wrapper, np.random.default_rng(21)
    k = 2 if activation == "tanh" else 1
    g = np.concatenate((np.linspace(-20, 20, 161), [-38.0, -30.0, 30.0, 38.0, 1e-3, -1e-3, 0.2499, 0.25, 0.0])).astype(np.float32)
    dim, rows = g.size, 1 if gate_rows == 0 else 3
    gate = np.broadcast_to(g, (rows, dim)) if gate_rows else g
    y, du = rng.normal(0, 1, (rows, dim)).astype(np.float32), rng.normal(0, 1, (rows, dim)).astype(np.float32)
    dgate, dx, dy = empty(w, gate.shape), empty(w, (rows, dim)), empty(w, (rows, dim))
    layer = normalization.BlockNorm(dim, "rms", None, residualScale=0.5, gateActivation=activation)
    layer.BackwardPropagation(dx, None, None, du=tensor(w, du), y=tensor(w, y), dy=dy, gate=tensor(w, gate), dGate=dgate, gateRows=gate_rows)
    e = np.exp(-k * np.abs(g.astype(np.float64)))
    want = 0.5 * du.astype(np.float64) * y * (k * k * e / (1 + e) ** 2)
    within(dgate.ToNumpy().reshape(want.shape), want, (16 + 2 * k * np.abs(g)) * ref.U * np.abs(want) + ref.TINY, "d_gate")


EXACT_ROWS = [(1, 5, None), (100, 60, 0), (4099, 64, 16), (3000, 100, 7), (5000, 128, 1), (2048, 512, 0), (1500, 516, 300), (6200, 700, 0),
              (4100, 1024, 2), (4150, 1023, 9), (6200, 1028, 0), (2500, 2044, 1000), (1030, 4096, 1), (600, 5001, 50), (1300, 8192, 0), (9000, 33, 4000)]


@pytest.mark.parametrize("rows,dim,gate_rows", EXACT_ROWS)
@pytest.mark.parametrize("stream,block", [("float32", "float32"), ("float32", "bfloat16"), ("bfloat16", "bfloat16")])
def test_block_norm_column_sums_lose_and_double_no_row(gpu_wrapper, rows, dim, gate_rows, stream, block):
    """Whole numbers all the way: mean 0 and 1 / deviation 1 as the statistics, weights and gates of 1 and 2, so that every
    term of the column sums is a whole number and every partial sum below 2^24 (2^8 for a gate's row in bf16): the formula's bits."""
    from sharpnet_amd import normalization
    w, rng = gpu_wrapper, np.random.default_rng(rows + dim)
    u, dh, y, du = (rng.integers(1, 4, (rows, dim)).astype(np.float32) for _ in range(4))
    sign = rng.choice([-1, 1], dim).astype(np.float32)
    dh, du = dh * sign, du * sign
    plain = np.tile(np.array([0, 1], np.float32), (rows, 1))
    gs = tensor(w, plain)
    weight = rng.choice([1, 2], dim).astype(np.float32)
    vec = lambda: empty(w, (dim,))  # noqa: E731
    # the norm ahead of the next block
    dx, dw, db = empty(w, (rows, dim), stream), vec(), vec()
    layer = normalization.BlockNorm(dim, "layer", "layer")
    dy = empty(w, (rows, dim), block)
    layer.BackwardPropagation(dx, tensor(w, u, stream), tensor(w, dh, block), y=tensor(w, y, block), dy=dy, postStatistics=gs, preStatistics=gs,
                              dPreWeight=dw, dPreBias=db)
    u64, dh64, y64, du64 = (a.astype(np.float64) for a in (u, dh, y, du))
    assert np.array_equal(dw.ToNumpy(), (dh64 * u64).sum(0)) and np.array_equal(db.ToNumpy(), dh64.sum(0))
    # the norm behind the block and its gate
    gate = None if gate_rows is None else rng.choice([1, 2], dim if gate_rows == 0 else (-(-rows // gate_rows), dim)).astype(np.float32)
    dpw, dpb, bias = vec(), vec(), np.ones(dim, np.float32)
    dgate = None if gate is None else empty(w, gate.shape, block if gate_rows else "float32")
    layer.BackwardPropagation(dx, None, None, du=tensor(w, du, stream), y=tensor(w, y, block), dy=dy, postStatistics=gs, postWeight=tensor(w, weight),
                              postBias=tensor(w, bias), dPostWeight=dpw, dPostBias=dpb, dGate=dgate, gateRows=gate_rows or 0,
                              gate=None if gate is None else tensor(w, gate, block if gate_rows else "float32"))
    t = du64
    if gate is not None:
        each = du64 * (y64 * weight + bias)
        if gate_rows == 0:
            assert np.array_equal(dgate.ToNumpy(), each.sum(0))
        else:
            want = np.zeros(gate.shape)
            np.add.at(want, np.arange(rows) // gate_rows, each)
            assert np.array_equal(dgate.ToNumpy().reshape(gate.shape), ref.bf16(want) if block == "bfloat16" else want)
        t = du64 * ref.gate_per_row(gate, gate_rows, rows, dim)
    assert np.array_equal(dpw.ToNumpy(), (t * y64).sum(0)) and np.array_equal(dpb.ToNumpy(), t.sum(0))
    assert np.array_equal(dx.ToNumpy().reshape(rows, dim), du)


@pytest.mark.parametrize("rows,dim,stream,block", [(70, 20, "float32", "float32"), (70, 61, "bfloat16", "bfloat16"), (40, 100, "float32", "bfloat16"),
                                                   (40, 127, "float32", "float32"), (20, 200, "bfloat16", "bfloat16"), (20, 510, "float32", "float32"),
                                                   (600, 700, "float32", "bfloat16"), (9, 1001, "float32", "float32"), (600, 1500, "bfloat16", "bfloat16"),
                                                   (5, 4096, "float32", "bfloat16"), (520, 5001, "float32", "float32"), (4, 8190, "bfloat16", "bfloat16")])
def test_block_norm_rows_that_are_not_finite_spoil_no_others(gpu_wrapper, rows, dim, stream, block):
    """NaN and infinities in a row, its gradients, statistics and gate: the other rows keep their bits."""
    from sharpnet_amd import normalization
    w, rng = gpu_wrapper, np.random.default_rng(dim)
    c = norm_case(rng, rows, dim, "layer", "rms", 1, True, stream, block)
    vectors = {k: tensor(w, v) for k, v in c["weights"].items()}
    du, dh = rounded(rng.normal(0, 1, (rows, dim)), stream), rounded(rng.normal(0, 1, (rows, dim)), block)
    layer = normalization.BlockNorm(dim, "layer", "rms", residualScale=0.7, gateActivation="tanh")
    bad = sorted({1, rows // 2, rows - 2})

    def results(spoil):
        host = {"x": c["x"].copy(), "y": c["y"].copy(), "gate": c["gate"].copy(), "du": du.copy(), "dh": dh.copy()}
        if spoil:
            for i, r in enumerate(bad):
                for k, name in enumerate(host):
                    host[name][r, (7 * k + i) % dim] = (np.nan, np.inf, -np.inf)[(i + k) % 3]
        x, y, gate, gdu, gdh = (tensor(w, host[k], stream if k in ("x", "du") else block) for k in host)
        out = {"u": empty(w, (rows, dim), stream), "h": empty(w, (rows, dim), block), "dx": empty(w, (rows, dim), stream),
               "dy": empty(w, (rows, dim), block), "dgate": empty(w, (rows, dim), block), "pre": empty(w, (rows, 2)), "post": empty(w, (rows, 2))}
        layer.ForwardPropagation(x, out["h"], y=y, u=out["u"], gate=gate, gateRows=1, preWeight=vectors["pre_weight"], preBias=vectors["pre_bias"],
                                 postWeight=vectors["post_weight"], postBias=vectors["post_bias"], preStatistics=out["pre"], postStatistics=out["post"])
        layer.BackwardPropagation(out["dx"], out["u"], gdh, du=gdu, y=y, dy=out["dy"], gate=gate, dGate=out["dgate"], gateRows=1,
                                  preWeight=vectors["pre_weight"], preStatistics=out["pre"], postWeight=vectors["post_weight"],
                                  postBias=vectors["post_bias"], postStatistics=out["post"])
        return {k: t.ToNumpy().reshape(rows, -1) for k, t in out.items()}
    clean, spoiled = results(False), results(True)
    others = np.setdiff1d(np.arange(rows), bad)
    for k in clean:
        assert np.all(np.isfinite(clean[k])), k
        assert np.array_equal(clean[k][others], spoiled[k][others]), k
        if k not in ("dgate", "post"):
            assert not np.any(np.all(np.isfinite(spoiled[k][bad]), axis=1)), k


def test_block_norm_rows_without_spread_and_missing_parts(gpu_wrapper):
    """Rows of one value (variance 0: 1 / deviation = 1 / sqrt(epsilon)), rows of zeros, a backward call without du and one
    without dh, gradients that are not wanted."""
    from sharpnet_amd import normalization
    w, rng = gpu_wrapper, np.random.default_rng(3)
    x = np.zeros((6, 36), np.float32)
    x[1], x[2], x[3] = 5.0, -1e4, rng.normal(1e3, 1, 36)
    gx = tensor(w, x)
    for kind in ("layer", "rms"):
        layer = normalization.BlockNorm(36, kind, None, epsilon=1e-5)
        h, s = empty(w, (6, 36)), empty(w, (6, 2))
        layer.ForwardPropagation(gx, h, preStatistics=s)
        want = ref.block_norm_forward(x, None, None, 0, kind, None, {}, 1.0, 1e-5, None, "float32", "float32")
        within(h.ToNumpy(), *want["h"], "h")
        within(s.ToNumpy(), *want["pre_statistics"], "statistics")
        dh = rng.normal(0, 1, (6, 36)).astype(np.float32)
        dx = empty(w, (6, 36))
        layer.BackwardPropagation(dx, gx, tensor(w, dh), preStatistics=s)
        back = ref.block_norm_backward(x, dh, None, None, None, 0, kind, None, {}, {"pre": s.ToNumpy()}, 1.0, None, "float32", "float32")
        within(dx.ToNumpy(), *back["dx"], "dx")
    # no dh: the gradients of the norm ahead of the next block are zeros, dy comes from du alone
    y, du = rng.normal(0, 1, (6, 36)).astype(np.float32), rng.normal(0, 1, (6, 36)).astype(np.float32)
    layer = normalization.BlockNorm(36, "rms", "layer", residualScale=2.0)
    stats = np.concatenate(ref.statistics(y, "layer", 1e-5), 1).astype(np.float32)
    dx, dy, dw, db, dpw = empty(w, (6, 36)), empty(w, (6, 36)), empty(w, (36,)), empty(w, (36,)), empty(w, (36,))
    layer.BackwardPropagation(dx, None, None, du=tensor(w, du), y=tensor(w, y), dy=dy, postStatistics=tensor(w, stats), dPreWeight=dw,
                              dPreBias=db, dPostWeight=dpw)
    back = ref.block_norm_backward(x, None, du, y, None, 0, "rms", "layer", {}, {"post": stats}, 2.0, None, "float32", "float32")
    assert np.array_equal(dx.ToNumpy(), du) and np.all(dw.ToNumpy() == 0) and np.all(db.ToNumpy() == 0)
    within(dy.ToNumpy(), *back["dy"], "dy")
    within(dpw.ToNumpy(), *back["d_post_weight"], "d_post_weight")


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("dim", [36, 260, 1001, 4096])
def test_block_norm_of_tiny_rows_without_epsilon(gpu_wrapper, kind, dim):
    """Rows whose mean square is below the normal numbers, epsilon = 0.  A square there and the mean are off by 2^-150 each
    besides their relative rounding: the variance by 2^-149 / variance, 1 / deviation by half of that."""
    from sharpnet_amd import normalization
    w, rng = gpu_wrapper, np.random.default_rng(dim)
    x = (rng.normal(0, 1, (5, dim)) * np.array([[1.0], [1e-18], [1e-19], [5e-20], [2e-20]])).astype(np.float32)
    h, s = empty(w, x.shape), empty(w, (5, 2))
    normalization.BlockNorm(dim, kind, epsilon=0.0).ForwardPropagation(tensor(w, x), h, preStatistics=s)
    mean, rstd = ref.statistics(x, kind, 0.0)
    rel = ref.C * ref.U + 2.0 ** -150 * rstd ** 2
    want = (x - mean) * rstd
    within(h.ToNumpy(), want, rel * (np.abs(x) + np.abs(x).mean(1, keepdims=True)) * rstd, "h")
    within(s.ToNumpy()[:, 1:], rstd, rel * rstd, "1 / deviation")


def test_block_norm_without_rows(gpu_wrapper):
    from sharpnet_amd import normalization
    w = gpu_wrapper
    layer = normalization.BlockNorm(8, "layer", "rms", gateActivation="sigmoid")
    none = lambda: tensor(w, np.zeros((0, 8)))  # noqa: E731
    layer.ForwardPropagation(none(), none(), y=none(), u=none(), gate=tensor(w, np.ones(8)))
    sums = [empty(w, (8,)) for _ in range(5)]
    layer.BackwardPropagation(none(), none(), none(), du=none(), y=none(), dy=none(), gate=tensor(w, np.ones(8)), dGate=sums[0],
                              dPreWeight=sums[1], dPreBias=sums[2], dPostWeight=sums[3], dPostBias=sums[4])
    for t in sums:
        assert np.all(t.ToNumpy() == 0)


def pitched(w, a, ld, offset, type_, fill=3.0):
    """a's rows at a pitch of ld elements, `offset` elements into a buffer."""
    whole = np.full((a.shape[0], ld), fill, np.float32)
    whole[:, :a.shape[1]] = a
    return tensor(w, np.concatenate((np.full(offset, fill, np.float32), whole.reshape(-1))), type_)


def rows_of(t, rows, dim, ld, offset, fill=3.0):
    got = t.ToNumpy()
    assert np.all(got[:offset] == fill)
    got = got[offset:].reshape(rows, ld)
    assert np.all(got[:, dim:] == fill)
    return got[:, :dim]


@pytest.mark.parametrize("dim,ld,offset", [(12, 20, 0), (12, 20, 4), (12, 21, 0), (12, 20, 1), (300, 301, 3), (1500, 1504, 4), (900, 903, 1), (700, 702, 3)])
def test_block_norm_rows_with_pitches_and_any_alignment(gpu_wrapper, dim, ld, offset):
    from sharpnet_amd.hiplib import ACT_SIGMOID, BlockNormDesc, NORM_LAYER, NORM_RMS, TYPES, check_status
    w, rng = gpu_wrapper, np.random.default_rng(ld)
    rows, stream, block = 21, "float32", "bfloat16"
    c = norm_case(rng, rows, dim, "layer", "rms", 4, True, stream, block)
    make = lambda a, t: pitched(w, a, ld, offset, t)  # noqa: E731
    at = lambda t: t.Pointer + t.ElementBytes * offset  # noqa: E731
    blank = np.full((rows, dim), 3.0, np.float32)
    x, y, gate, u, h = make(c["x"], stream), make(c["y"], block), make(c["gate"], block), make(blank, stream), make(blank, block)
    vec = {k: tensor(w, v) for k, v in c["weights"].items()}
    pre_s, post_s = empty(w, (rows, 2)), empty(w, (rows, 2))
    d = BlockNormDesc(stream_type=TYPES[stream], block_type=TYPES[block], pre_norm=NORM_LAYER, post_norm=NORM_RMS,
                      gate_activation=ACT_SIGMOID, dim=dim, gate_rows=4, rows=rows, ld_x=ld, ld_y=ld, ld_u=ld, ld_h=ld, ld_gate=ld,
                      epsilon=1e-5, residual_scale=0.7, x=at(x), y=at(y), u=at(u), h=at(h), gate=at(gate),
                      pre_statistics=pre_s.Pointer, post_statistics=post_s.Pointer, **{k: v.Pointer for k, v in vec.items()})
    check_status(w.lib.snhip_block_norm_forward(w.handle, ctypes.byref(d)))
    want = ref.block_norm_forward(c["x"], c["y"], c["gate"], 4, "layer", "rms", c["weights"], 0.7, 1e-5, "sigmoid", stream, block)
    within(rows_of(u, rows, dim, ld, offset), *want["u"], "u")
    within(rows_of(h, rows, dim, ld, offset), *want["h"], "h")
    du, dh = rng.normal(0, 1, (rows, dim)).astype(np.float32), rounded(rng.normal(0, 1, (rows, dim)), block)
    gdu, gdh, dx, dy = make(du, stream), make(dh, block), make(blank, stream), make(blank, block)
    dgate = make(blank[:6], block)
    sums = {k: empty(w, (dim,)) for k in ("d_pre_weight", "d_pre_bias", "d_post_weight", "d_post_bias")}
    d.du, d.dh, d.dx, d.dy, d.d_gate = at(gdu), at(gdh), at(dx), at(dy), at(dgate)
    for k, v in sums.items():
        setattr(d, k, v.Pointer)
    need = ctypes.c_size_t()
    check_status(w.lib.snhip_block_norm_backward_workspace_size(ctypes.byref(d), ctypes.byref(need)))
    ws = empty(w, [need.value], "uint8")
    check_status(w.lib.snhip_block_norm_backward(w.handle, ctypes.byref(d), ws.Pointer, need.value))
    stats = {"pre": pre_s.ToNumpy(), "post": post_s.ToNumpy()}
    back = ref.block_norm_backward(rows_of(u, rows, dim, ld, offset), dh, du, c["y"], c["gate"], 4, "layer", "rms", c["weights"], stats, 0.7,
                                   "sigmoid", stream, block)
    within(rows_of(dx, rows, dim, ld, offset), *back["dx"], "dx")
    within(rows_of(dy, rows, dim, ld, offset), *back["dy"], "dy")
    within(rows_of(dgate, 6, dim, ld, offset), *back["d_gate"], "d_gate")
    for k, v in sums.items():
        within(v.ToNumpy(), *back[k], k)


# ---------------------------------------------------------------------------------------------------------------
# AdamW
# ---------------------------------------------------------------------------------------------------------------
ADAM = dict(learningRate=0.01, beta1=0.9, beta2=0.99, epsilon=1e-6)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("gradients", ["float32", "bfloat16"])
@pytest.mark.parametrize("offset", [0, 1])
def test_adamw(gpu_wrapper, bits, gradients, offset):
    """Tensors of all kinds of sizes in one buffer each for parameters and gradients (at any element offset), three steps:
    the moments bit for bit (states in 8 bits: every code and scale), the parameters within their bound, the copies as the
    rounded parameters, the gaps between the tensors as they were."""
    from sharpnet_amd import GPUTensor, optimizer
    w, rng = gpu_wrapper, np.random.default_rng(bits + offset)
    sizes = [1, 3, 4, 255, 256, 257, 0, 4095, 4096, 4097, 10001]
    at, total = [], offset
    for n in sizes:
        at.append(total)
        total += n + (4 - n % 4 if offset == 0 else 5)
    p = rng.normal(0, 1, total).astype(np.float32)
    g = rounded(rng.normal(0, 1, total) * np.exp(rng.normal(-3, 4, total)), gradients)
    g[rng.integers(0, total, total // 10)] = 0
    gp, gg, gc = tensor(w, p), tensor(w, g, gradients), tensor(w, np.full(total, 3.0, np.float32), "bfloat16")
    cut = lambda t: [t.Slice(a, [n]) for a, n in zip(at, sizes)]  # noqa: E731
    copies = [c if k % 2 == 0 else None for k, c in enumerate(cut(gc))]
    decay = [0.1 * (k % 3) for k in range(len(sizes))]
    opt = optimizer.AdamW(cut(gp), cut(gg), weightDecay=decay, stateBits=bits, seed=2 ** 33 + 5, copies=copies, **ADAM)
    now = p.copy()
    state = [(np.zeros(n, np.float32), np.zeros(n, np.float32)) for n in sizes]
    for step in (1, 2, 3):
        scale = 0.5 if step == 2 else 1.0
        opt.Step(gradientScale=scale)
        got = gp.ToNumpy()
        inside = np.zeros(total, bool)
        for k, (a, n) in enumerate(zip(at, sizes)):
            inside[a:a + n] = True
            if n == 0:
                continue
            m, v = ref.moments(state[k][0], state[k][1], g[a:a + n] * np.float32(scale), 0.9, 0.99)
            new, bound = ref.new_parameters(now[a:a + n], m, v, 0.01, decay[k], 0.9, 0.99, 1e-6, step)
            within(got[a:a + n], new, bound, "p of tensor %d, step %d" % (k, step))
            if bits == 32:
                assert np.array_equal(opt.States[k][0].ToNumpy(), m) and np.array_equal(opt.States[k][1].ToNumpy(), v), (k, step)
                state[k] = m, v
            else:
                words = ref.random_words(n, k, step, 2 ** 33 + 5)
                (mc, ms), (vc, vs) = ref.store_m(m, words), ref.store_v(v, words)
                for t, want in zip(opt.States[k], (mc, vc, ms, vs)):
                    assert np.array_equal(t.ToNumpy(), want), (k, step)
                state[k] = ref.load8(mc, ms, ref.E4M3), ref.load8(vc, vs, ref.E5M2)
        assert np.array_equal(got[~inside], p[~inside])
        now = got
    copy = gc.ToNumpy()
    for k, (a, n) in enumerate(zip(at, sizes)):
        want = ref.bf16(now[a:a + n]) if k % 2 == 0 else np.full(n, 3.0)
        assert np.array_equal(copy[a:a + n], want), k
    opt.Dispose()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_gradients_that_are_not_finite_or_at_the_ends_of_the_range(gpu_wrapper, bits):
    """NaN and infinities spoil their own element alone; denormal, tiny and huge gradients keep to the definition."""
    from sharpnet_amd import GPUTensor, optimizer
    w, rng = gpu_wrapper, np.random.default_rng(8)
    n = 1024
    g = rng.normal(0, 1, n).astype(np.float32)
    g[[0, 300, 301, 700]] = [np.nan, np.inf, -np.inf, np.nan]
    g[256:512] *= np.float32(1e-20)      # v below the normal numbers
    g[512:768] *= np.float32(1e17)
    g[768:] = 0
    gp, gg = tensor(w, np.ones(n, np.float32)), tensor(w, g)
    opt = optimizer.AdamW([gp], [gg], weightDecay=0.0, stateBits=bits, seed=4, **ADAM)
    z = np.zeros(n, np.float32)
    m, v = z, z
    p = np.ones(n, np.float32)
    for step in (1, 2):
        opt.Step()
        m, v = ref.moments(m, v, g, 0.9, 0.99)
        ok = np.isfinite(m) & np.isfinite(v)
        got = gp.ToNumpy()
        new, bound = ref.new_parameters(p[ok], m[ok], v[ok], 0.01, 0.0, 0.9, 0.99, 1e-6, step)
        within(got[ok], new, bound, "p")
        if bits == 32:
            assert np.array_equal(opt.States[0][0].ToNumpy(), m, equal_nan=True) and np.array_equal(opt.States[0][1].ToNumpy(), v, equal_nan=True)
        else:
            words = ref.random_words(n, 0, step, 4)
            (mc, ms), (vc, vs) = ref.store_m(m, words), ref.store_v(v, words)
            for t, want in zip(opt.States[0], (mc, vc, ms, vs)):
                assert np.array_equal(t.ToNumpy(), want), step
            m, v = ref.load8(mc, ms, ref.E4M3), ref.load8(vc, vs, ref.E5M2)
        p = got


def test_adamw_8_bit_v_is_never_zero_beside_a_huge_one(gpu_wrapper):
    """A block's elements of 1e-20 beside one of 1e32: what scaling by the block's power of two leaves of them is below the
    smallest fp32 number, stored they are the smallest code, not zero."""
    from sharpnet_amd import optimizer
    w, n = gpu_wrapper, 600
    g = np.zeros(n, np.float32)
    g[0], g[1], g[2:200:3], g[256:512], g[512] = 1e17, 1e-9, -1e-9, 1e-9, 1e17
    opt = optimizer.AdamW([tensor(w, np.ones(n, np.float32))], [tensor(w, g)], weightDecay=0.0, stateBits=8, seed=4, **ADAM)
    opt.Step()
    z = np.zeros(n, np.float32)
    m, v = ref.moments(z, z, g, 0.9, 0.99)
    code, scale = ref.store_v(v, ref.random_words(n, 0, 1, 4))
    assert np.array_equal(opt.States[0][3].ToNumpy(), scale)
    below = (v > 0) & (v * np.repeat(ref.power(127 - scale.astype(np.int64)), 256)[:n] == 0)
    assert below.sum() == 67
    assert np.array_equal(opt.States[0][1].ToNumpy(), np.where(below, 1, code))


def test_adamw_of_memory_that_has_gone(gpu_wrapper):
    """Parameters that are parts of one buffer: the step is refused once the buffer is disposed, not for a view of it."""
    from sharpnet_amd import optimizer
    w = gpu_wrapper
    whole, grads = tensor(w, np.ones(300)), tensor(w, np.ones(300))
    views = [whole.Slice(0, [100]), whole.Slice(100, [10, 20])]
    opt = optimizer.AdamW(views, [grads.Slice(0, [100]), grads.Slice(100, [10, 20])])
    opt.Step()
    views[0].Dispose()
    opt.Step()
    before = whole.ToNumpy().copy()
    assert np.all(before[:300] < 1)
    whole.Dispose()
    with pytest.raises(RuntimeError):
        opt.Step()
    assert opt.StepCount == 2


def test_adamw_8_bit_states_follow_a_slow_mean(gpu_wrapper):
    """beta2 = 0.999 moves v by a thousandth of its distance a step, a hundredth of a step of e5m2.  From v = 0 and gradients
    of 1 the mean of v over n elements is 1 - 0.999^t; rounding at random keeps it: the rounding of a step moves an element
    by at most one step of its binade, 1/4 v, with mean 0 and a standard deviation of at most 1/8 v (and a block's largest
    element, below whose binade the others stay, changes no values).  After t steps the mean of n elements is off by at most
    5 sqrt(t) / 8 / sqrt(n) v with a probability of 6e-7; the generator's words are a fixed function of the seed."""
    from sharpnet_amd import optimizer
    w, n, steps = gpu_wrapper, 65536, 60
    gp, gg = tensor(w, np.zeros(n, np.float32)), tensor(w, np.ones(n, np.float32))
    opt = optimizer.AdamW([gp], [gg], learningRate=0.0, beta1=0.9, beta2=0.999, stateBits=8, seed=11)
    for _ in range(steps):
        opt.Step()
    v = ref.load8(opt.States[0][1].ToNumpy(), opt.States[0][3].ToNumpy(), ref.E5M2).astype(np.float64)
    m = ref.load8(opt.States[0][0].ToNumpy(), opt.States[0][2].ToNumpy(), ref.E4M3).astype(np.float64)
    want = 1 - 0.999 ** steps
    assert abs(v.mean() - want) <= 5 * np.sqrt(steps) / 8 / np.sqrt(n) * want + 2.0 ** -16 * want * steps
    want = 1 - 0.9 ** steps
    assert abs(m.mean() - want) <= 5 * np.sqrt(steps) / 16 / np.sqrt(n) * want + 2.0 ** -16 * want * steps


# ---------------------------------------------------------------------------------------------------------------
# streams, graphs
# ---------------------------------------------------------------------------------------------------------------
def step_of_everything(w, rng, wrapper_of_workspaces=None):
    """Tensors of one pass through all the operators, and the function that runs it."""
    from sharpnet_amd import embedding, normalization, optimizer
    tokens, vocabulary, dim = 900, 400, 96
    x = tensor(w, make_ids(rng, tokens, vocabulary, "int32"), "int32")
    table, dW = tensor(w, rng.normal(0, 1, (vocabulary, dim))), empty(w, (vocabulary, dim))
    e = embedding.WordEmbedding(vocabulary, dim, 2.0)
    s, y, u, h = (empty(w, (tokens, dim)) for _ in range(4))
    y = tensor(w, rng.normal(0, 1, (tokens, dim)))
    gate = tensor(w, rng.normal(0, 1, dim))
    ps, qs = empty(w, (tokens, 2)), empty(w, (tokens, 2))
    wt, dwt, dgate = tensor(w, rng.normal(1, 0.1, dim)), empty(w, (dim,)), empty(w, (dim,))
    dx, dy, dh = empty(w, (tokens, dim)), empty(w, (tokens, dim)), tensor(w, rng.normal(0, 1, (tokens, dim)))
    n = normalization.BlockNorm(dim, "rms", "layer", gateActivation="sigmoid")
    opt = optimizer.AdamW([table, wt], [dW, dwt], stateBits=8, seed=3)

    def work():
        e.ForwardPropagation(s, x, table)
        n.ForwardPropagation(s, h, y=y, u=u, gate=gate, preWeight=wt, preStatistics=ps, postStatistics=qs)
        n.BackwardPropagation(dx, u, dh, y=y, dy=dy, gate=gate, dGate=dgate, preWeight=wt, preStatistics=ps, dPreWeight=dwt, postStatistics=qs)
        e.BackwardPropagation(dW, x, dx)

    return work, (s, u, h, ps, qs, dx, dy, dgate, dwt, dW), opt


def hip_runtime():
    hip = ctypes.CDLL("libamdhip64.so")
    vp = ctypes.c_void_p
    for name, args in (("hipStreamBeginCapture", [vp, ctypes.c_int]), ("hipStreamEndCapture", [vp, ctypes.POINTER(vp)]),
                       ("hipGraphInstantiate", [ctypes.POINTER(vp), vp, vp, vp, ctypes.c_size_t]),
                       ("hipGraphLaunch", [vp, vp]), ("hipGraphExecDestroy", [vp]), ("hipGraphDestroy", [vp])):
        getattr(hip, name).argtypes = args
        getattr(hip, name).restype = ctypes.c_int
    return hip


def test_training_operators_under_graph_capture(gpu_wrapper):
    """Forward, backward and an AdamW step captured once and replayed: each replay gives what the eager calls give."""
    from sharpnet_amd.hiplib import check_status
    w = gpu_wrapper
    work, outs, opt = step_of_everything(w, np.random.default_rng(1))
    work()                                   # eager: also sizes the layers' scratch memory
    w.synchronize()
    eager = [t.ToNumpy().copy() for t in outs]
    reference, _, other = step_of_everything(w, np.random.default_rng(1))
    reference()
    hip, vp = hip_runtime(), ctypes.c_void_p
    stream, graph, graph_exec = vp(), vp(), vp()
    check_status(w.lib.snhip_stream_create(ctypes.byref(stream)), "snhip_stream_create")
    check_status(w.lib.snhip_set_stream(w.handle, stream), "snhip_set_stream")
    try:
        assert hip.hipStreamBeginCapture(stream, 0) == 0
        try:
            work()
            opt.Step()
        finally:
            assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(graph_exec), graph, None, None, 0) == 0
        for rep in range(3):
            for t in outs:
                t.SetValue(float("nan"))
            table = other.Parameters[0].ToNumpy()
            assert np.array_equal(opt.Parameters[0].ToNumpy(), table), rep
            w.synchronize()
            assert hip.hipGraphLaunch(graph_exec, stream) == 0
            w.synchronize()
            if rep == 0:
                for t, want in zip(outs, eager):
                    assert np.array_equal(t.ToNumpy(), want)
            # eager on the twin: the captured step's scalars are those of step 1 in every replay
            reference()
            other.StepCount = 0
            other.Step()
            for a, b in zip(opt.Parameters + sum(opt.States, []), other.Parameters + sum(other.States, [])):
                assert np.array_equal(a.ToNumpy(), b.ToNumpy()), rep
    finally:
        check_status(w.lib.snhip_set_stream(w.handle, None), "snhip_set_stream")
        if graph_exec:
            hip.hipGraphExecDestroy(graph_exec)
        if graph:
            hip.hipGraphDestroy(graph)
        check_status(w.lib.snhip_stream_destroy(stream), "snhip_stream_destroy")


def test_training_operators_on_two_streams_at_once(gpu_wrapper):
    """Two handles on two streams, calls in turn without waiting: scratch memory is each caller's own."""
    from sharpnet_amd import GPUWrapper
    from sharpnet_amd.hiplib import check_status
    want = []
    for seed in (5, 6):
        work, outs, _ = step_of_everything(gpu_wrapper, np.random.default_rng(seed))
        work()
        want.append([t.ToNumpy().copy() for t in outs])
    wrappers, streams, jobs = [GPUWrapper(0), GPUWrapper(0)], [], []
    for w, seed in zip(wrappers, (5, 6)):
        s = ctypes.c_void_p()
        check_status(w.lib.snhip_stream_create(ctypes.byref(s)))
        streams.append(s)
        jobs.append(step_of_everything(w, np.random.default_rng(seed)))
        jobs[-1][0]()
        w.synchronize()
        check_status(w.lib.snhip_set_stream(w.handle, s))
    for _ in range(10):
        for work, _, _ in jobs:
            work()
    for w in wrappers:
        w.synchronize()
    for w, s, (_, outs, opt), expected in zip(wrappers, streams, jobs, want):
        for t, value in zip(outs, expected):
            assert np.array_equal(t.ToNumpy(), value)
        opt.Dispose()
        check_status(w.lib.snhip_set_stream(w.handle, None))
        check_status(w.lib.snhip_stream_destroy(s))


def test_launches_of_more_workgroups_than_a_grid_row(gpu_wrapper):
    """Launches of over 65536 workgroups are spread over two dimensions of the grid: inputs that repeat every few rows give
    outputs that do, bit for bit."""
    from sharpnet_amd import embedding, normalization, optimizer
    w, rng = gpu_wrapper, np.random.default_rng(8)
    # one row of 520 elements to a workgroup of 256 threads, four in turn
    tokens, dim, period = 4 * 65536 + 4 * 8 + 3, 520, 71
    W = rounded(rng.normal(0, 1, (period, dim)), "bfloat16")
    y = empty(w, (tokens, dim), "bfloat16")
    embedding.WordEmbedding(period, dim).ForwardPropagation(y, tensor(w, (np.arange(tokens) % period).astype(np.int32), "int32"),
                                                            tensor(w, W, "bfloat16"))
    y = y.ToNumpy().reshape(tokens, dim)
    for k in range(0, tokens, period):
        assert np.array_equal(y[k:k + period], W[:tokens - k]), k
    del y
    # four rows of 68 elements to a workgroup
    rows, dim, period = 4 * 65536 + 1, 68, 64
    x = np.resize(rng.normal(0, 1, (period, dim)).astype(np.float32), (rows, dim))
    h, first = empty(w, (rows, dim)), empty(w, (period, dim))
    layer = normalization.BlockNorm(dim, "layer")
    layer.ForwardPropagation(tensor(w, x), h)
    layer.ForwardPropagation(tensor(w, x[:period]), first)
    h, first = h.ToNumpy(), first.ToNumpy()
    assert np.all(np.isfinite(first)) and np.array_equal(h, np.resize(first, (rows, dim)))
    # 1024 elements to a workgroup
    sizes = [65535 * 1024 + 5, 3, 2048]
    short = [2048, 3, 2048]
    g = rng.normal(0, 1, 2048).astype(np.float32)
    result = []
    for lengths in (sizes, short):
        parameters = [tensor(w, np.resize(np.float32(0.5) * g, n)) for n in lengths]
        opt = optimizer.AdamW(parameters, [tensor(w, np.resize(g, n)) for n in lengths], **ADAM)
        opt.Step()
        result.append([t.ToNumpy() for tensors in [parameters] + opt.States for t in tensors])
        opt.Dispose()
    for a, b in zip(*result):
        assert np.array_equal(a, np.resize(b, a.size))


def test_scratch_memory_that_has_grown_after_a_capture(gpu_wrapper):
    """A graph goes on using the scratch memory it was captured with when a longer batch has come along."""
    from sharpnet_amd import embedding
    from sharpnet_amd.hiplib import check_status
    w, rng = gpu_wrapper, np.random.default_rng(9)
    hip, vp = hip_runtime(), ctypes.c_void_p
    layer = embedding.WordEmbedding(300, 40)

    def batch(tokens):
        x, dy = make_ids(rng, tokens, 300, "int32"), rng.normal(0, 1, (tokens, 40)).astype(np.float32)
        return tensor(w, x, "int32"), tensor(w, dy), empty(w, (300, 40))
    x, dy, dW = batch(5000)
    layer.BackwardPropagation(dW, x, dy)
    want = dW.ToNumpy().copy()
    stream, graph, graph_exec = vp(), vp(), vp()
    check_status(w.lib.snhip_stream_create(ctypes.byref(stream)), "snhip_stream_create")
    check_status(w.lib.snhip_set_stream(w.handle, stream), "snhip_set_stream")
    try:
        assert hip.hipStreamBeginCapture(stream, 0) == 0
        try:
            layer.BackwardPropagation(dW, x, dy)
        finally:
            assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(graph_exec), graph, None, None, 0) == 0
        for tokens in (9000, 30000):
            longer = batch(tokens)
            layer.BackwardPropagation(longer[2], longer[0], longer[1])
            other = empty(w, (2 << 20,))  # where freed memory would go
            dW.SetValue(float("nan"))
            assert hip.hipGraphLaunch(graph_exec, stream) == 0
            w.synchronize()
            assert np.array_equal(dW.ToNumpy(), want), tokens
            assert np.all(np.isnan(other.ToNumpy()))
    finally:
        check_status(w.lib.snhip_set_stream(w.handle, None), "snhip_set_stream")
        if graph_exec:
            hip.hipGraphExecDestroy(graph_exec)
        if graph:
            hip.hipGraphDestroy(graph)
        check_status(w.lib.snhip_stream_destroy(stream), "snhip_stream_destroy")
        layer.Dispose()


def test_embedding_gradients_with_scratch_memory_on_two_handles_at_once(gpu_wrapper):
    """Long batches of two handles on two streams in turn, one layer: whole numbers, so the formula's bits (one token lost or read
    from the other batch would show)."""
    from sharpnet_amd import GPUWrapper, embedding
    from sharpnet_amd.hiplib import check_status
    rng, vocabulary, dim = np.random.default_rng(15), 2000, 24
    layer, jobs = embedding.WordEmbedding(vocabulary, dim, 2.0), []
    for tokens in (50000, 8200):
        w, stream = GPUWrapper(0), ctypes.c_void_p()
        check_status(w.lib.snhip_stream_create(ctypes.byref(stream)))
        x, dy = make_ids(rng, tokens, vocabulary, "int64"), rng.integers(-8, 9, (tokens, dim)).astype(np.float32)
        jobs.append((w, stream, tensor(w, x, "int64"), tensor(w, dy), empty(w, (vocabulary, dim)), ref.embedding_backward(x, dy, vocabulary, 2.0)[0]))
        w.synchronize()
        check_status(w.lib.snhip_set_stream(w.handle, stream))
    for _ in range(3):
        for _ in range(10):
            for w, _, x, dy, dW, _ in jobs:
                layer.BackwardPropagation(dW, x, dy)
        for w, _, _, _, dW, want in jobs:
            assert np.array_equal(dW.ToNumpy(), want)
            dW.SetValue(float("nan"))
            w.synchronize()
    for w, stream, *_ in jobs:
        check_status(w.lib.snhip_set_stream(w.handle, None))
        check_status(w.lib.snhip_stream_destroy(stream))
    layer.Dispose()


def test_one_layer_on_two_streams_of_a_handle(gpu_wrapper):
    """Gradients of a long and a short batch in turn on two streams of one handle, without waiting: each stream's calls have
    scratch memory of their own (the sums of a call do not depend on the other's).  Then the same under a capture on a stream
    that the layers have not been used on, replayed beside eager calls."""
    from sharpnet_amd import embedding, normalization
    from sharpnet_amd.hiplib import check_status
    w, rng = gpu_wrapper, np.random.default_rng(12)
    hip, vp = hip_runtime(), ctypes.c_void_p
    vocabulary, dim = 3000, 64
    e, n = embedding.WordEmbedding(vocabulary, dim), normalization.BlockNorm(dim, "rms")

    def job(tokens):
        x, dy = tensor(w, make_ids(rng, tokens, vocabulary, "int32"), "int32"), tensor(w, rng.normal(0, 1, (tokens, dim)))
        s = tensor(w, np.concatenate(ref.statistics(dy.ToNumpy(), "rms", 1e-5), 1))
        dW, dx, dw = empty(w, (vocabulary, dim)), empty(w, (tokens, dim)), empty(w, (dim,))

        def work():
            e.BackwardPropagation(dW, x, dy)
            n.BackwardPropagation(dx, dy, dy, preStatistics=s, dPreWeight=dw)
        return work, (dW, dx, dw)
    jobs = [job(40000), job(9000)]
    want = []
    for work, outs in jobs:
        work()
        want.append([t.ToNumpy().copy() for t in outs])

    def check():
        for (_, outs), expected in zip(jobs, want):
            for t, value in zip(outs, expected):
                assert np.array_equal(t.ToNumpy(), value)
                t.SetValue(float("nan"))
        w.synchronize()
    streams, graph, graph_exec = [vp(), vp(), vp()], vp(), vp()
    for s in streams:
        check_status(w.lib.snhip_stream_create(ctypes.byref(s)), "snhip_stream_create")
    try:
        for _ in range(4):
            for _ in range(5):
                for (work, _), s in zip(jobs, streams):
                    check_status(w.lib.snhip_set_stream(w.handle, s), "snhip_set_stream")
                    work()
            for s in streams[:2]:
                check_status(w.lib.snhip_set_stream(w.handle, s), "snhip_set_stream")
                w.synchronize()
            check()
        check_status(w.lib.snhip_set_stream(w.handle, streams[2]), "snhip_set_stream")
        assert hip.hipStreamBeginCapture(streams[2], 0) == 0
        try:
            jobs[0][0]()
        finally:
            assert hip.hipStreamEndCapture(streams[2], ctypes.byref(graph)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(graph_exec), graph, None, None, 0) == 0
        for _ in range(4):
            check_status(w.lib.snhip_set_stream(w.handle, streams[1]), "snhip_set_stream")
            for _ in range(3):
                jobs[1][0]()
                assert hip.hipGraphLaunch(graph_exec, streams[2]) == 0
            for s in streams[1:]:
                check_status(w.lib.snhip_set_stream(w.handle, s), "snhip_set_stream")
                w.synchronize()
            check()
    finally:
        check_status(w.lib.snhip_set_stream(w.handle, None), "snhip_set_stream")
        if graph_exec:
            hip.hipGraphExecDestroy(graph_exec)
        if graph:
            hip.hipGraphDestroy(graph)
        for s in streams:
            check_status(w.lib.snhip_stream_destroy(s), "snhip_stream_destroy")
        e.Dispose()
        n.Dispose()


# ---------------------------------------------------------------------------------------------------------------
# together, as a training step uses them
# ---------------------------------------------------------------------------------------------------------------
def test_a_training_step_of_a_small_network(gpu_wrapper):
    """Embedding, norm, multi-head attention, join with gate, Dense with ReLU, join, output projection; backward through all
    of it; AdamW on every parameter.  Against torch's autograd on the CPU in 64 bits.

    Bound: every stage is off by at most 64 u (4e-6) of its magnitudes; products here sum at most 64 terms and the bar of the
    Dot path is 1e-4 sqrt(K) of the largest operands, 8e-4 at K = 64 (it holds them to a few u in practice).  Gradients pass
    some twenty stages: 20 x 4e-6 x an amplification of at most 4 in these well-scaled layers gives 3.2e-4 of the tensor's
    largest gradient."""
    import torch
    from sharpnet_amd import GPUTensor, attention, embedding, linear, normalization, optimizer
    w, rng = gpu_wrapper, np.random.default_rng(7)
    B, T, V, D, H, F = 3, 16, 50, 32, 4, 64
    ids = rng.integers(0, V, (B, T)).astype(np.int32)
    ids[2, 11:] = -1                                    # a shorter sequence
    host = {"table": rng.normal(0, 1 / np.sqrt(D), (V, D)), "n1": rng.normal(1, 0.1, D), "n2": rng.normal(1, 0.1, D),
            "b2": rng.normal(0, 0.1, D), "p1": rng.normal(1, 0.1, D), "gate": rng.normal(0, 1, D), "n3": rng.normal(1, 0.1, D),
            "wq": rng.normal(0, 1 / np.sqrt(D), (D, D)), "wk": rng.normal(0, 1 / np.sqrt(D), (D, D)), "wv": rng.normal(0, 1 / np.sqrt(D), (D, D)),
            "wo": rng.normal(0, 1 / np.sqrt(D), (D, D)), "w1": rng.normal(0, 1 / np.sqrt(D), (F, D)), "f1": rng.normal(0, 0.1, F),
            "w2": rng.normal(0, 1 / np.sqrt(F), (D, F)), "out": rng.normal(0, 1 / np.sqrt(D), (V, D))}
    host = {k: v.astype(np.float32) for k, v in host.items()}
    dlogits = rng.normal(0, 1, (B * T, V)).astype(np.float32)
    dlogits[ids.reshape(-1) < 0] = 0

    # the oracle
    P = {k: torch.tensor(v.astype(np.float64), requires_grad=True) for k, v in host.items()}
    keep = torch.tensor((ids >= 0).astype(np.float64))[..., None]
    rms = lambda z, g: z / torch.sqrt((z * z).mean(-1, keepdim=True) + 1e-5) * g  # noqa: E731
    norm = lambda z, g, b: (z - z.mean(-1, keepdim=True)) / torch.sqrt(z.var(-1, unbiased=False, keepdim=True) + 1e-5) * g + b  # noqa: E731
    x0 = P["table"][torch.tensor(np.maximum(ids, 0)).long()] * keep * float(np.float32(np.sqrt(D)))
    h0 = rms(x0, P["n1"])
    split = lambda z: z.reshape(B, T, H, D // H).transpose(1, 2)  # noqa: E731
    q, k, v = (split(h0 @ P[n].T) for n in ("wq", "wk", "wv"))
    s = (q @ k.transpose(2, 3)) / np.sqrt(D // H)
    s = s.masked_fill(torch.triu(torch.ones(T, T, dtype=torch.bool), 1), -1e12)
    a = (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(B, T, D) @ P["wo"].T
    x1 = x0 + 0.5 * torch.sigmoid(P["gate"]) * rms(a, P["p1"])
    h1 = norm(x1, P["n2"], P["b2"])
    f = torch.relu(h1 @ P["w1"].T + P["f1"]) @ P["w2"].T
    x2 = x1 + f
    logits = rms(x2, P["n3"]) @ P["out"].T
    (logits.reshape(B * T, V) * torch.tensor(dlogits.astype(np.float64))).sum().backward()

    # the network
    G = {k: tensor(w, v) for k, v in host.items()}
    dG = {k: empty(w, v.shape) for k, v in host.items()}
    new = lambda *shape: GPUTensor(list(shape), None, w)  # noqa: E731
    emb = embedding.WordEmbedding(V, D, np.sqrt(D))
    first, join1, join2 = (normalization.BlockNorm(D, "rms"), normalization.BlockNorm(D, "layer", "rms", 0.5, "sigmoid"),
                           normalization.BlockNorm(D, "rms"))
    gids = tensor(w, ids, "int32")
    X0, H0, A, X1, H1, F1, F2, X2, H2, L = (new(B, T, n) for n in (D, D, D, D, D, F, D, D, D, V))
    S0, S1, SP, S2 = (new(B * T, 2) for _ in range(4))
    emb.ForwardPropagation(X0, gids, G["table"])
    first.ForwardPropagation(X0, H0, preWeight=G["n1"], preStatistics=S0)
    state = attention.MultiheadAttentionForwardPropagation(H0, H0, H0, A, G["wq"], G["wk"], G["wv"], G["wo"], H, D // H, D // H, is_causal=True)
    join1.ForwardPropagation(X0, H1, y=A, u=X1, gate=G["gate"], preWeight=G["n2"], preBias=G["b2"], postWeight=G["p1"], preStatistics=S1,
                             postStatistics=SP)
    linear.DenseForwardPropagation(F1, H1, G["w1"], G["f1"], True, activation="CUDNN_ACTIVATION_RELU")
    linear.DenseForwardPropagation(F2, F1, G["w2"], None, True)
    join2.ForwardPropagation(X1, H2, y=F2, u=X2, preWeight=G["n3"], preStatistics=S2)
    linear.DenseForwardPropagation(L, H2, G["out"], None, True)

    def near(got, want, name):
        assert np.max(np.abs(got.reshape(want.shape) - want)) <= 3.2e-4 * np.max(np.abs(want)), name
    near(L.ToNumpy(), logits.detach().numpy(), "logits")
    dL = tensor(w, dlogits).Reshape(B, T, V)
    dH2, dX1, dF2, dF1, dH1, dX0, dA = (new(B, T, n) for n in (D, D, D, F, D, D, D))
    dense = dict(compatibility_mode="PyTorch", flattenInputTensorOnLastDimension=True)
    linear.DenseBackwardPropagation(dH2, dG["out"], None, H2, dL, G["out"], **dense)
    join2.BackwardPropagation(dX1, X2, dH2, y=F2, dy=dF2, preWeight=G["n3"], preStatistics=S2, dPreWeight=dG["n3"])
    linear.DenseBackwardPropagation(dF1, dG["w2"], None, F1, dF2, G["w2"], **dense)
    F1.ActivationBackward("CUDNN_ACTIVATION_RELU", 0.0, dF1, dF1)
    linear.DenseBackwardPropagation(dH1, dG["w1"], dG["f1"], H1, dF1, G["w1"], **dense)
    join1.BackwardPropagation(dX0, X1, dH1, du=dX1, y=A, dy=dA, gate=G["gate"], dGate=dG["gate"], preWeight=G["n2"], preStatistics=S1,
                              dPreWeight=dG["n2"], dPreBias=dG["b2"], postWeight=G["p1"], postStatistics=SP, dPostWeight=dG["p1"])
    dQ, dK, dV = (new(B, T, D) for _ in range(3))
    grads = {n: (dG[g], None) for n, g in (("w_Q", "wq"), ("w_K", "wk"), ("w_V", "wv"), ("out_proj_weight", "wo"))}
    attention.MultiheadAttentionBackwardPropagation(dQ, dK, dV, H0, H0, H0, dA, state, G["wq"], G["wk"], G["wv"], G["wo"], grads)
    dQ.Update_Adding_Alpha_X(1.0, dK)
    dQ.Update_Adding_Alpha_X(1.0, dV)
    first.BackwardPropagation(dX0, X0, dQ, du=dX0, preWeight=G["n1"], preStatistics=S0, dPreWeight=dG["n1"])
    emb.BackwardPropagation(dG["table"], gids, dX0)
    for n in host:
        near(dG[n].ToNumpy(), P[n].grad.numpy(), "gradient of " + n)
    names = sorted(host)
    opt = optimizer.AdamW([G[n] for n in names], [dG[n] for n in names], learningRate=0.01, weightDecay=0.1)
    given = {n: dG[n].ToNumpy() for n in names}
    opt.Step()
    for n in names:
        z = np.zeros_like(host[n])
        m, v = ref.moments(z, z, given[n], 0.9, 0.999)
        want, bound = ref.new_parameters(host[n], m, v, 0.01, 0.1, 0.9, 0.999, 1e-8, 1)
        within(G[n].ToNumpy(), want, bound, n)
