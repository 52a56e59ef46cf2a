"""Word embedding, block norm and AdamW without a GPU: descriptor layouts, refusals (all before any device work), and the
plain forms that the GPU tests compare with: their gradients against differences, their 8-bit formats against torch's,
their random words against the published vectors."""
import ctypes

import numpy as np
import pytest

from sharpnet_amd import hiplib
from tests import training_reference as ref

S = hiplib.CublasStatus
OK_SO_FAR = S.CUBLAS_STATUS_NOT_INITIALIZED   # the arguments were taken; there is no device to go on with
BAD, UNSUPPORTED = S.CUBLAS_STATUS_INVALID_VALUE, S.CUBLAS_STATUS_NOT_SUPPORTED


@pytest.fixture
def lib():
    import torch
    if torch.cuda.is_available():
        pytest.skip("checks what happens on a machine without a GPU")
    return hiplib.load_library()


@pytest.fixture
def handle():
    """Something that is not NULL; its device cannot be made current here, so no call gets past its argument checks."""
    return ctypes.addressof(_HANDLE)


_HANDLE = ctypes.create_string_buffer(4096)
A = 0x10000000          # an address like any other (aligned, never touched)


def test_descriptor_layouts(lib):
    assert lib.snhip_sizeof_embedding_desc() == ctypes.sizeof(hiplib.EmbeddingDesc)
    assert lib.snhip_sizeof_block_norm_desc() == ctypes.sizeof(hiplib.BlockNormDesc)
    assert lib.snhip_sizeof_adamw_tensor() == ctypes.sizeof(hiplib.AdamwTensor)
    assert lib.snhip_sizeof_adamw_step_desc() == ctypes.sizeof(hiplib.AdamwStepDesc)
    for cls in (hiplib.EmbeddingDesc, hiplib.BlockNormDesc, hiplib.AdamwStepDesc):
        with pytest.raises(TypeError):
            cls(no_such_field=1)


EMBEDDING = dict(id_type=hiplib.TYPE_I32, table_type=hiplib.TYPE_F32, output_type=hiplib.TYPE_BF16, tokens=10, vocabulary=7, dim=6)


@pytest.mark.parametrize("change,status", [
    ({}, OK_SO_FAR), ({"ld_table": 6, "ld_output": 9}, OK_SO_FAR), ({"padding_index": 100}, OK_SO_FAR),
    ({"struct_size": 4}, BAD), ({"id_type": hiplib.TYPE_BF16}, BAD), ({"id_type": 9}, BAD), ({"table_type": hiplib.TYPE_I32}, BAD),
    ({"output_type": -1}, BAD), ({"tokens": -1}, BAD), ({"vocabulary": -1}, BAD), ({"dim": -1}, BAD), ({"ld_table": 5}, BAD),
    ({"ld_output": 5}, BAD), ({"padding_index": -2}, BAD), ({"tokens": 2 ** 31}, UNSUPPORTED)])
def test_embedding_descriptor_checks(lib, handle, change, status):
    d = hiplib.EmbeddingDesc(**{**EMBEDDING, **change})
    n = ctypes.c_size_t()
    assert lib.snhip_embedding_forward(handle, ctypes.byref(d), A, A, A) == status
    assert lib.snhip_embedding_backward(handle, ctypes.byref(d), A, A, A, 0, A, 1 << 40) == status
    assert lib.snhip_embedding_backward_workspace_size(ctypes.byref(d), ctypes.byref(n)) == (0 if status == OK_SO_FAR else status)


def test_embedding_pointer_checks(lib, handle):
    d = hiplib.EmbeddingDesc(**EMBEDDING)
    r, n = ctypes.byref(d), ctypes.c_size_t()
    assert lib.snhip_embedding_forward(None, r, A, A, A) == S.CUBLAS_STATUS_NOT_INITIALIZED
    assert lib.snhip_embedding_forward(handle, None, A, A, A) == BAD
    for args in ((None, A, A), (A, None, A), (A, A, None), (A + 2, A, A), (A, A + 2, A), (A, A, A + 1)):
        assert lib.snhip_embedding_forward(handle, r, *args) == BAD, args
    assert lib.snhip_embedding_backward_workspace_size(r, None) == BAD
    # few tokens: no scratch memory
    assert lib.snhip_embedding_backward_workspace_size(r, ctypes.byref(n)) == 0 and n.value == 0
    assert lib.snhip_embedding_backward(handle, r, A, A, A, 0, None, 0) == OK_SO_FAR
    d.tokens = 5000
    assert lib.snhip_embedding_backward_workspace_size(r, ctypes.byref(n)) == 0 and n.value > 0
    full = n.value
    for args in ((None, A, A, 0, A, full), (A, None, A, 0, A, full), (A, A, None, 0, A, full), (A, A, A, 0, None, full),
                 (A, A, A, 0, A + 4, full), (A, A, A, 0, A, full - 1), (A, A + 1, A, 0, A, full), (A, A, A + 2, 0, A, full)):
        assert lib.snhip_embedding_backward(handle, r, *args) == BAD, args
    assert lib.snhip_embedding_backward(handle, r, A, A, A, 0, A, full) == OK_SO_FAR
    d.tokens = 0      # nothing to look up, nothing to add
    assert lib.snhip_embedding_forward(handle, r, None, None, None) == 0
    assert lib.snhip_embedding_backward(handle, r, None, None, None, 1, None, 0) == 0
    assert lib.snhip_embedding_backward(handle, r, None, None, None, 0, None, 0) == BAD   # the gradient has to be cleared
    d.id_type, d.tokens = hiplib.TYPE_I64, 4
    assert lib.snhip_embedding_forward(handle, r, A + 4, A, A) == BAD


NORM = dict(stream_type=hiplib.TYPE_F32, block_type=hiplib.TYPE_BF16, pre_norm=hiplib.NORM_LAYER, post_norm=hiplib.NORM_RMS,
            gate_activation=hiplib.ACT_SIGMOID, dim=12, gate_rows=3, rows=10, x=A, y=A, u=A, h=A, gate=A, pre_statistics=A,
            post_statistics=A, du=A, dh=A, dx=A, dy=A)


@pytest.mark.parametrize("change,forward,backward", [
    ({}, OK_SO_FAR, OK_SO_FAR), ({"gate_rows": 0}, OK_SO_FAR, OK_SO_FAR), ({"dim": 8192}, OK_SO_FAR, OK_SO_FAR),
    ({"struct_size": 8}, BAD, BAD), ({"stream_type": hiplib.TYPE_I32}, BAD, BAD), ({"block_type": 7}, BAD, BAD),
    ({"pre_norm": 3}, BAD, BAD), ({"post_norm": -1}, BAD, BAD), ({"gate_activation": hiplib.ACT_RELU}, UNSUPPORTED, UNSUPPORTED),
    ({"rows": -1}, BAD, BAD), ({"dim": -4}, BAD, BAD), ({"gate_rows": -1}, BAD, BAD), ({"ld_x": 11}, BAD, BAD), ({"ld_gate": 1}, BAD, BAD),
    ({"epsilon": -1.0}, BAD, BAD), ({"epsilon": float("nan")}, BAD, BAD), ({"epsilon": float("inf")}, BAD, BAD),
    ({"dim": 8193}, UNSUPPORTED, UNSUPPORTED), ({"rows": 2 ** 31}, UNSUPPORTED, UNSUPPORTED),
    ({"stream_type": hiplib.TYPE_BF16, "block_type": hiplib.TYPE_F32}, UNSUPPORTED, UNSUPPORTED),
    ({"y": None}, BAD, BAD), ({"y": None, "gate": None}, BAD, BAD), ({"y": None, "gate": None, "post_norm": 0}, OK_SO_FAR, OK_SO_FAR),
    ({"y": None, "gate": None, "post_norm": 0, "pre_norm": 0}, BAD, BAD),
    ({"x": None}, BAD, OK_SO_FAR), ({"u": None}, BAD, BAD), ({"h": None}, BAD, OK_SO_FAR), ({"dx": None}, OK_SO_FAR, BAD),
    ({"dy": None}, OK_SO_FAR, BAD), ({"dh": None}, OK_SO_FAR, OK_SO_FAR), ({"du": None}, OK_SO_FAR, OK_SO_FAR),
    ({"du": None, "dh": None}, OK_SO_FAR, BAD), ({"pre_norm": 0}, OK_SO_FAR, BAD), ({"pre_norm": 0, "dh": None}, OK_SO_FAR, OK_SO_FAR),
    ({"pre_statistics": None}, OK_SO_FAR, BAD), ({"post_statistics": None}, OK_SO_FAR, BAD),
    ({"gate": None, "d_gate": A}, OK_SO_FAR, BAD), ({"x": A + 2}, BAD, BAD), ({"y": A + 1}, BAD, BAD), ({"gate": A + 1}, BAD, BAD),
    ({"gate": A + 2, "gate_rows": 0}, BAD, BAD), ({"pre_weight": A + 2}, BAD, BAD), ({"d_post_bias": A + 1}, BAD, BAD)])
def test_block_norm_checks(lib, handle, change, forward, backward):
    d = hiplib.BlockNormDesc(**{**NORM, **change})
    assert lib.snhip_block_norm_forward(handle, ctypes.byref(d)) == forward
    n = ctypes.c_size_t()
    assert lib.snhip_block_norm_backward_workspace_size(ctypes.byref(d), ctypes.byref(n)) == (0 if backward == OK_SO_FAR else backward)
    assert lib.snhip_block_norm_backward(handle, ctypes.byref(d), A, 1 << 40) == backward


def test_block_norm_workspace_and_handle_checks(lib, handle):
    d = hiplib.BlockNormDesc(**{**NORM, "d_pre_weight": A, "d_gate": A, "gate_rows": 0})
    r, n = ctypes.byref(d), ctypes.c_size_t()
    assert lib.snhip_block_norm_forward(None, r) == lib.snhip_block_norm_backward(None, r, A, 1 << 40) == S.CUBLAS_STATUS_NOT_INITIALIZED
    assert lib.snhip_block_norm_forward(handle, None) == lib.snhip_block_norm_backward(handle, None, A, 1 << 40) == BAD
    assert lib.snhip_block_norm_backward_workspace_size(r, None) == BAD
    assert lib.snhip_block_norm_backward_workspace_size(r, ctypes.byref(n)) == 0 and n.value > 0
    for ws, size in ((None, n.value), (A + 8, n.value), (A, n.value - 1)):
        assert lib.snhip_block_norm_backward(handle, r, ws, size) == BAD
    assert lib.snhip_block_norm_backward(handle, r, A, n.value) == OK_SO_FAR
    d.d_pre_weight = d.d_gate = None      # nothing to sum up: no scratch memory
    assert lib.snhip_block_norm_backward_workspace_size(r, ctypes.byref(n)) == 0 and n.value == 0
    assert lib.snhip_block_norm_backward(handle, r, None, 0) == OK_SO_FAR
    d.rows = 0
    assert lib.snhip_block_norm_forward(handle, r) == 0


def adamw_tensors(*changes):
    made = (hiplib.AdamwTensor * len(changes))()
    for k, (t, change) in enumerate(zip(made, changes)):
        base = A + (k << 20)
        fields = dict(parameter=base, gradient=base + 0x10000, moment1=base + 0x20000, moment2=base + 0x30000, scale1=base + 0x40000,
                      scale2=base + 0x50000, bf16_copy=base + 0x60000, count=1000, gradient_type=hiplib.TYPE_F32, weight_decay=0.1)
        for f, v in {**fields, **change}.items():
            setattr(t, f, v)
    return made


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("change,status", [
    ({}, OK_SO_FAR), ({"bf16_copy": None}, OK_SO_FAR), ({"count": 0, "parameter": None}, 0), ({"count": -1}, BAD),
    ({"parameter": None}, BAD), ({"gradient": None}, BAD), ({"moment1": None}, BAD), ({"moment2": None}, BAD),
    ({"parameter": A + 2}, BAD), ({"gradient": A + 0x10001}, BAD), ({"bf16_copy": A + 0x60001}, BAD), ({"gradient_type": hiplib.TYPE_I32}, BAD),
    ({"weight_decay": float("nan")}, BAD), ({"moment2": A + 0x20000}, BAD), ({"bf16_copy": A + 2000}, BAD), ({"gradient": A}, BAD),
    ({"gradient": A + 3996}, BAD), ({"gradient": A + 4000}, OK_SO_FAR)])
def test_adamw_plan_checks(lib, handle, bits, change, status):
    plan = ctypes.c_void_p(1)
    assert lib.snhip_adamw_create(handle, adamw_tensors(change), 1, bits, ctypes.byref(plan)) == \
        (status if status != 0 else OK_SO_FAR)
    assert not plan.value


def test_adamw_scales_several_tensors_and_arguments(lib, handle):
    plan = ctypes.c_void_p()
    create = lambda t, n, bits: lib.snhip_adamw_create(handle, t, n, bits, ctypes.byref(plan))  # noqa: E731
    assert create(adamw_tensors({"scale1": None}), 1, 8) == BAD and create(adamw_tensors({"scale1": None}), 1, 32) == OK_SO_FAR
    assert create(adamw_tensors({"scale2": A + 0x40003}), 1, 8) == BAD      # four blocks: bytes 0 to 3 are scale1's
    assert create(adamw_tensors({"scale2": A + 0x40004}), 1, 8) == OK_SO_FAR
    assert create(adamw_tensors({}, {}), 2, 8) == OK_SO_FAR
    assert create(adamw_tensors({}, {"parameter": A}), 2, 32) == BAD        # the same tensor twice
    assert create(adamw_tensors({}, {"parameter": A + 4000}), 2, 32) == OK_SO_FAR
    assert create(adamw_tensors({}, {"gradient": A + 0x10000}), 2, 32) == OK_SO_FAR   # gradients are only read
    assert create(adamw_tensors({}), 1, 16) == UNSUPPORTED
    assert create(adamw_tensors({"count": 2 ** 62}), 1, 32) == create(adamw_tensors({"count": 2 ** 63 - 1}), 1, 8) == UNSUPPORTED
    assert create(adamw_tensors({"count": 2 ** 40}, {"count": 2 ** 40}), 2, 8) == UNSUPPORTED   # 2^31 chunks
    assert create(None, 1, 32) == BAD and create(adamw_tensors({}), -1, 32) == BAD
    assert lib.snhip_adamw_create(handle, None, 0, 32, None) == BAD
    assert lib.snhip_adamw_create(None, None, 0, 32, ctypes.byref(plan)) == S.CUBLAS_STATUS_NOT_INITIALIZED
    assert lib.snhip_adamw_destroy(None) == 0


@pytest.mark.parametrize("change", [{"struct_size": 8}, {"step": 0}, {"step": -3}, {"learning_rate": float("nan")}, {"beta1": 1.0}, {"beta1": -0.1},
                                    {"beta2": 1.0}, {"beta2": float("nan")}, {"epsilon": -1e-8}, {"epsilon": float("inf")},
                                    {"gradient_scale": float("inf")}])
def test_adamw_step_checks(lib, handle, change):
    plan = ctypes.create_string_buffer(256)      # a plan of no chunks on device 0
    d = hiplib.AdamwStepDesc(learning_rate=1e-3)
    assert lib.snhip_adamw_step(handle, ctypes.addressof(plan), ctypes.byref(d)) == 0
    assert lib.snhip_adamw_step(handle, None, ctypes.byref(d)) == lib.snhip_adamw_step(None, ctypes.addressof(plan), ctypes.byref(d)) == \
        S.CUBLAS_STATUS_NOT_INITIALIZED
    for k, v in change.items():
        setattr(d, k, v)
    assert lib.snhip_adamw_step(handle, ctypes.addressof(plan), ctypes.byref(d)) == BAD
    assert lib.snhip_adamw_step(handle, ctypes.addressof(plan), None) == BAD


@pytest.mark.parametrize("change,status", [({"epsilon": 1e-40}, BAD), ({"epsilon": 1e-300}, BAD), ({"epsilon": 0.0}, 0), ({"epsilon": 2.0 ** -126}, 0),
                                           ({"learning_rate": 1e39}, BAD), ({"learning_rate": -1e39}, BAD), ({"learning_rate": 1e38}, BAD),
                                           ({"learning_rate": 1e38, "beta1": 0.0}, 0), ({"learning_rate": 0.0}, 0)])
def test_adamw_scalars_that_fp32_does_not_hold(lib, handle, change, status):
    """1e38 / (1 - 0.9) is beyond fp32's largest number; an epsilon below its normal numbers would be a division by zero."""
    plan = ctypes.create_string_buffer(256)      # a plan of no chunks on device 0
    d = hiplib.AdamwStepDesc(**{"learning_rate": 1e-3, **change})
    assert lib.snhip_adamw_step(handle, ctypes.addressof(plan), ctypes.byref(d)) == status


class Stub:
    """Shape and type of a tensor, for the host side's checks."""
    _disposed, _owner, handle = False, None, None

    def __init__(self, shape, type_="float32", device=0):
        self.Shape, self.Type, self.Pointer, self.device_id = list(shape), type_, A, device
        self.Count = int(np.prod(shape))
        self.lib = self._lib = self.Wrapper = self

    def AssertIsNotDisposed(self):
        pass

    def __getattr__(self, name):  # as a library: calls that nothing was refused of
        if not name.startswith("snhip_"):
            raise AttributeError(name)
        return lambda *args: 0


def test_host_sides_refuse_what_does_not_fit():
    from sharpnet_amd import GPUTensor, embedding, normalization, optimizer
    e = embedding.WordEmbedding(7, 6)
    ids, y, table = Stub((10,), "int32"), Stub((10, 6)), Stub((7, 6))
    for args in ((Stub((9, 6)), ids, table), (Stub((10, 5)), ids, table), (y, ids, Stub((6, 6))), (y, Stub((10,), "uint8"), table),
                 (Stub((10, 6), "int32"), ids, table), (y, ids, Stub((7, 6), "int64"))):
        with pytest.raises(ValueError):
            e.ForwardPropagation(*args)
    with pytest.raises(ValueError):
        e.BackwardPropagation(Stub((7, 6), "bfloat16"), ids, y)
    with pytest.raises(ValueError):
        embedding.WordEmbedding(-1, 6)
    with pytest.raises(ValueError):
        normalization.BlockNorm(8, "batch")
    with pytest.raises(hiplib.SharpNetHipError):
        normalization.BlockNorm(8, gateActivation="CUDNN_ACTIVATION_RELU")
    n = normalization.BlockNorm(8, "layer", "rms")
    x, h, y = Stub((5, 8)), Stub((5, 8)), Stub((5, 8))
    for kw in (dict(y=Stub((4, 8))), dict(y=Stub((5, 8), "bfloat16")), dict(u=Stub((5, 8), "bfloat16")), dict(preWeight=Stub((7,))),
               dict(preWeight=Stub((8,), "bfloat16")), dict(preStatistics=Stub((5,))), dict(gate=Stub((8,)), gateRows=2),
               dict(gate=Stub((3, 8)), gateRows=0), dict(gate=Stub((8,)), gateRows=-1)):
        with pytest.raises(ValueError):
            n.ForwardPropagation(x, h, **{**dict(y=y, u=Stub((5, 8))), **kw})
    with pytest.raises(ValueError):
        n.BackwardPropagation(x, x, h, y=y, dy=y, gate=Stub((8,)), dGate=Stub((8, 1)))
    p, g = Stub((3, 4)), Stub((3, 4))
    good = [[Stub((3, 4)), Stub((3, 4))]]
    for kw in (dict(parameters=[Stub((3, 4), "bfloat16")]), dict(gradients=[Stub((3, 5))]), dict(gradients=[]), dict(copies=[Stub((3, 4))]),
               dict(stateBits=16), dict(stateBits=8), dict(states=[[Stub((3, 4))]]), dict(weightDecay=[0.1, 0.2])):
        with pytest.raises(ValueError):
            optimizer.AdamW(**{**dict(parameters=[p], gradients=[g], states=good), **kw})
    with pytest.raises(ValueError):
        GPUTensor.FromPointer([4], A + 2, "float32", gpu_wrapper=p)
    t = GPUTensor.FromPointer([4], A + 2, "bfloat16", gpu_wrapper=p, owner=ids)
    assert t.ElementBytes == 2 and t.Slice(1, [2]).Pointer == A + 4 and t.Slice(1, [2]).Type == "bfloat16" and not t.IsOwnerOfMemory


def test_host_sides_refuse_tensors_of_another_device():
    from sharpnet_amd import embedding, normalization, optimizer
    e, n = embedding.WordEmbedding(7, 6), normalization.BlockNorm(6, "rms")
    ids, y, table, far = Stub((10,), "int32"), Stub((10, 6)), Stub((7, 6)), Stub((7, 6), device=1)
    for call in (lambda: e.ForwardPropagation(y, ids, far), lambda: e.BackwardPropagation(far, ids, y),
                 lambda: n.ForwardPropagation(y, Stub((10, 6), device=1)), lambda: n.BackwardPropagation(y, Stub((10, 6), device=1), y),
                 lambda: optimizer.AdamW([table], [far], states=[[table, table]])):
        with pytest.raises(ValueError, match="device 1"):
            call()


def test_entry_points_that_compute_with_float32_refuse_other_types():
    from sharpnet_amd import GPUTensor, attention, linear
    w = Stub((1,))
    new = lambda type_, *shape: GPUTensor.FromPointer(list(shape), A, type_, gpu_wrapper=w)  # noqa: E731
    f, b = new("float32", 4, 4), new("bfloat16", 4, 4)
    f3, b3, v = new("float32", 2, 4, 4), new("bfloat16", 2, 4, 4), new("int32", 4)
    for call in (lambda: f.Dot(f, False, b, False), lambda: b.Dot(f, f), lambda: f3.BatchMatrixMultiplication(b3, False, f3, False, 1.0, 0.0),
                 lambda: f.DotRowMajor(f, False, f, False, 1.0, 0.0, bias=v), lambda: f.GemmEx(A=b, B=f), lambda: f.GemmEx(A=b, B=f, bias=b, math=2),
                 lambda: b.Compute_BiasGradient_from_dy(new("float32", 4)), lambda: f.Update_Adding_Alpha_X(1.0, b),
                 lambda: b.SoftmaxLastDimension(f), lambda: f.Transpose(b), lambda: f.ActivationForward("CUDNN_ACTIVATION_RELU", 0.0, b),
                 lambda: b.SetValue(1.0), lambda: linear.DenseForwardPropagation(f, f, b, None, False),
                 lambda: attention.fused_attention_forward(f3, f3, b3, f3, None, batch=2, heads=1, tq=4, tkv=4, dk=4, dv=4, scale=1.0,
                                                           is_causal=False, packed=False)):
        with pytest.raises(ValueError, match="float32"):
            call()
    assert f.FloatPointer == f.Pointer == A


def test_one_layer_called_by_two_threads():
    """Every call's descriptor is its own, whatever another thread asks of the layer meanwhile."""
    import threading
    import time
    from sharpnet_amd import embedding, normalization
    e, n, wrong = embedding.WordEmbedding(7, 6), normalization.BlockNorm(6, "rms"), []

    def run(rows):
        def check(handle, d, *args):
            time.sleep(1e-4)
            got = d._obj.tokens if isinstance(d._obj, hiplib.EmbeddingDesc) else d._obj.rows
            if got != rows:
                wrong.append((got, rows))
            return 0
        y, ids, table = Stub((rows, 6)), Stub((rows,), "int32"), Stub((7, 6))
        y.snhip_embedding_forward = y.snhip_block_norm_forward = check
        for _ in range(100):
            e.ForwardPropagation(y, ids, table)
            n.ForwardPropagation(y, Stub((rows, 6)))
    threads = [threading.Thread(target=run, args=(rows,)) for rows in (3, 4, 5)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_layers_that_are_changed_between_calls():
    """The next call goes by the norms, the activation and the sizes that the layer has by then, its scratch size included."""
    from sharpnet_amd import embedding, normalization
    seen, sizes = [], []
    kind = lambda d: (d.pre_norm, d.post_norm, d.gate_activation, d.dim, d.epsilon, d.residual_scale)  # noqa: E731

    def tensor(*shape, type_="float32"):
        t = Stub(shape, type_)
        t.snhip_block_norm_forward = t.snhip_block_norm_backward = lambda handle, d, *rest: seen.append(kind(d._obj)) or 0
        t.snhip_block_norm_backward_workspace_size = lambda d, out: sizes.append(kind(d._obj)) or 0
        t.snhip_embedding_forward = lambda handle, d, *rest: seen.append((d._obj.vocabulary, d._obj.dim)) or 0
        return t
    n = normalization.BlockNorm(8, "layer", "rms", 0.5, epsilon=0.25)
    x, v, s = tensor(5, 8), tensor(8), tensor(5, 2)

    def both(x, v):
        n.ForwardPropagation(x, x, y=x, u=x, gate=v, preWeight=v)
        n.BackwardPropagation(x, x, x, y=x, dy=x, gate=v, preWeight=v, preStatistics=s, postStatistics=s)
        return seen[-2:], sizes[-1:]
    want = (hiplib.NORM_LAYER, hiplib.NORM_RMS, hiplib.ACT_NONE, 8, 0.25, 0.5)
    assert both(x, v) == ([want] * 2, [want])
    n.PreNorm, n.PostNorm, n.GateActivation, n.Epsilon, n.ResidualScale = hiplib.NORM_RMS, hiplib.NORM_LAYER, hiplib.ACT_TANH, 0.5, 2.0
    want = (hiplib.NORM_RMS, hiplib.NORM_LAYER, hiplib.ACT_TANH, 8, 0.5, 2.0)
    assert both(x, v) == ([want] * 2, [want])
    n.EmbeddingDim = 4
    with pytest.raises(ValueError):
        both(x, v)
    with pytest.raises(ValueError):
        both(tensor(10, 4), v)
    s = tensor(10, 2)
    assert both(tensor(10, 4), tensor(4))[0] == [want[:3] + (4,) + want[4:]] * 2
    e = embedding.WordEmbedding(7, 6)
    e.ForwardPropagation(tensor(10, 6), tensor(10, type_="int32"), tensor(7, 6))
    e.VocabularySize = 9
    with pytest.raises(ValueError):
        e.ForwardPropagation(tensor(10, 6), tensor(10, type_="int32"), tensor(7, 6))
    e.ForwardPropagation(tensor(10, 6), tensor(10, type_="int32"), tensor(9, 6))
    assert seen[-2:] == [(7, 6), (9, 6)]


def test_sizes_beyond_32_bits_are_not_cut_off():
    """Numbers that the descriptors' 32-bit fields do not hold: refused, or what they mean where they mean something."""
    from sharpnet_amd import embedding, normalization, optimizer
    seen = []

    def tensor(*shape, type_="float32"):
        t = Stub(shape, type_)
        t.snhip_embedding_forward = lambda handle, d, *rest: seen.append((d._obj.vocabulary, d._obj.dim, d._obj.padding_index)) or 0
        t.snhip_block_norm_forward = lambda handle, d: seen.append(d._obj.gate_rows) or 0
        t.snhip_adamw_step = lambda handle, plan, d: seen.append(d._obj.step) or 0
        return t
    large, ids = 2 ** 32 + 5, tensor(10, type_="int32")
    for vocabulary, dim in ((large, 1), (7, large), (2 ** 31, 1)):
        with pytest.raises(ValueError):
            embedding.WordEmbedding(vocabulary, dim).ForwardPropagation(tensor(10, dim), ids, tensor(vocabulary, dim))
    for padding in (large, 2 ** 31, 2 ** 32 - 1, 7):  # beyond the vocabulary: no token's
        embedding.WordEmbedding(7, 6, paddingIndex=padding).ForwardPropagation(tensor(10, 6), ids, tensor(7, 6))
    embedding.WordEmbedding(7, 6, paddingIndex=6).ForwardPropagation(tensor(10, 6), ids, tensor(7, 6))
    assert seen == [(7, 6, -1)] * 4 + [(7, 6, 6)]
    seen.clear()
    with pytest.raises(ValueError):
        normalization.BlockNorm(large).ForwardPropagation(tensor(1, large), tensor(1, large))
    x = tensor(10, 6)
    for rows in (2 ** 32, large, 2 ** 31):  # one row of the gate for all
        normalization.BlockNorm(6).ForwardPropagation(x, x, y=x, u=x, gate=tensor(1, 6), gateRows=rows)
    assert seen == [2 ** 31 - 1] * 3
    seen.clear()
    opt = optimizer.AdamW([x], [x], states=[[x, x]], step=2 ** 31 - 2)
    opt._plan = ctypes.c_void_p(A)
    opt.Step()
    for opt.StepCount in (2 ** 31 - 1, 2 ** 32, large):
        with pytest.raises(ValueError):
            opt.Step()
    assert seen == [2 ** 31 - 1]
    opt._plan = None


def test_block_norm_outputs_that_would_stay_as_they_are_are_refused():
    from sharpnet_amd import normalization
    x, s = Stub((5, 8)), Stub((5, 2))
    norm, join, bare = normalization.BlockNorm(8), normalization.BlockNorm(8, None, "rms"), normalization.BlockNorm(8, None)
    for call in (lambda: norm.ForwardPropagation(x, x, u=x), lambda: join.ForwardPropagation(x, x, y=x, u=x),
                 lambda: bare.ForwardPropagation(x, x, y=x, u=x), lambda: norm.BackwardPropagation(x, x, x, dy=x, preStatistics=s),
                 lambda: bare.BackwardPropagation(x, None, None, du=x, dy=x),
                 lambda: join.ForwardPropagation(x, None, y=x, u=x, preStatistics=s), lambda: norm.ForwardPropagation(x, x, postStatistics=s)):
        with pytest.raises(ValueError):
            call()
    norm.ForwardPropagation(x, x, preStatistics=s)
    join.ForwardPropagation(x, None, y=x, u=x, postStatistics=s)
    bare.BackwardPropagation(x, None, None, du=x, y=x, dy=x)


def test_layers_call_the_wrapper_they_are_made_for():
    from sharpnet_amd import embedding, normalization
    used, own, far = [], Stub((1,)), Stub((1,), device=1)
    own.handle = "own"

    def tensor(*shape, type_="float32"):
        t = Stub(shape, type_)
        t.handle = "tensor's"
        for name in ("embedding_forward", "embedding_backward", "block_norm_forward", "block_norm_backward"):
            setattr(t, "snhip_" + name, lambda handle, *rest: used.append(handle) or 0)
        return t
    x, ids, table = tensor(10, 6), tensor(10, type_="int32"), tensor(7, 6)

    def calls(w):
        e, n = embedding.WordEmbedding(7, 6, gpu_wrapper=w), normalization.BlockNorm(6, gpu_wrapper=w)
        return (lambda: e.ForwardPropagation(x, ids, table), lambda: e.BackwardPropagation(table, ids, x), lambda: n.ForwardPropagation(x, x),
                lambda: n.BackwardPropagation(x, x, x, preStatistics=tensor(10, 2)))
    for w, handle in ((own, "own"), (None, "tensor's")):
        for call in calls(w):
            call()
        assert used == [handle] * 4
        used.clear()
    for call in calls(far):
        with pytest.raises(ValueError, match="device 1"):
            call()


def test_workspace_of_a_layer():
    """One for each wrapper; a longer one leaves the one before in place until Dispose."""
    from sharpnet_amd.gpu_tensor import LayerWorkspace

    class Wrapper:
        def __init__(self):
            self.lib, self.live = None, []

        def allocate(self, nbytes):
            self.live.append(nbytes)
            return A + len(self.live)

        def release(self, pointer, nbytes):
            self.live.remove(nbytes)

    a, b, held = Wrapper(), Wrapper(), LayerWorkspace()
    assert held.Get(a, 0) is None and not a.live
    first = held.Get(a, 1000)
    assert held.Get(a, 800) is first and held.Get(b, 800) is not first
    second = held.Get(a, 1001)
    assert second.Count == 1500 and not first._disposed and a.live == [1000, 1500] and b.live == [800]
    held.Dispose()
    assert first._disposed and second._disposed and not a.live and not b.live


def test_scratch_memory_goes_by_stream(lib, handle):
    """Calls on two streams of one handle may overlap: each has its own scratch memory, the same one when it comes again."""
    from sharpnet_amd import embedding, normalization
    stream, allocated, given = [0], [], []

    class Wrapper:
        lib, device_id, handle = None, 0, None

        def allocate(self, nbytes):
            allocated.append(nbytes)
            return A + (len(allocated) << 24)

        def release(self, pointer, nbytes):
            pass

        def snhip_get_stream(self, handle, out):
            out._obj.value = stream[0]
            return 0

        def snhip_embedding_backward_workspace_size(self, desc, out):
            return lib.snhip_embedding_backward_workspace_size(desc, out)

        def snhip_block_norm_backward_workspace_size(self, desc, out):
            return lib.snhip_block_norm_backward_workspace_size(desc, out)

        def snhip_embedding_backward(self, handle, desc, ids, dy, table, accumulate, workspace, nbytes):
            given.append(workspace)
            return 0

        def snhip_block_norm_backward(self, handle, desc, workspace, nbytes):
            given.append(workspace)
            return 0
    w = Wrapper()
    w.lib = w

    def on(shape, type_="float32"):
        t = Stub(shape, type_)
        t.Wrapper = t._lib = w
        return t
    e, n = embedding.WordEmbedding(7, 6), normalization.BlockNorm(6, "rms")
    ids, dy, dW, stats, dw = on((9000,), "int32"), on((9000, 6)), on((7, 6)), on((9000, 2)), on((6,))
    for call in (lambda: e.BackwardPropagation(dW, ids, dy),
                 lambda: n.BackwardPropagation(dy, dy, dy, preStatistics=stats, dPreWeight=dw)):
        given.clear()
        for stream[0] in (0, 0x1000, 0x2000, 0x1000, 0):
            call()
        null, first, second = given[:3]
        assert len({null, first, second}) == 3 and None not in given and given[3:] == [first, null]
    p, q = ctypes.c_void_p(1), ctypes.byref(ctypes.c_void_p())
    assert lib.snhip_get_stream(None, q) == S.CUBLAS_STATUS_NOT_INITIALIZED and lib.snhip_get_stream(handle, None) == BAD
    assert lib.snhip_get_stream(handle, ctypes.byref(p)) == 0 and not p.value


def test_one_layers_scratch_memory_in_two_threads():
    """Two threads, each with a handle of its own: gradients of one layer never get the other's scratch memory, whatever their sizes."""
    import threading
    import time
    from sharpnet_amd import embedding, normalization
    e, n, wrong = embedding.WordEmbedding(7, 6), normalization.BlockNorm(6, "rms"), []

    class Wrapper:
        device_id = 0

        def __init__(self, number):
            self.lib, self.handle, self.base, self.made = self, number, A * (1 + number), 0

        def allocate(self, nbytes):
            time.sleep(1e-4)
            self.made += 1
            return self.base + (self.made << 12)

        def release(self, pointer, nbytes):
            pass

        def snhip_get_stream(self, handle, out):
            time.sleep(1e-4)
            out._obj.value = 0x1000 * handle
            return 0

        def size(self, desc, out):
            time.sleep(1e-4)
            out._obj.value = (desc._obj.tokens if isinstance(desc._obj, hiplib.EmbeddingDesc) else desc._obj.rows) * 4
            return 0
        snhip_embedding_backward_workspace_size = snhip_block_norm_backward_workspace_size = size

        def check(self, rows, pointer, nbytes):
            if not self.base <= pointer < self.base + A or nbytes < 4 * rows:
                wrong.append((self.handle, rows, pointer, nbytes))
            return 0

        def snhip_embedding_backward(self, handle, desc, ids, dy, table, accumulate, workspace, nbytes):
            return self.check(desc._obj.tokens, workspace, nbytes)

        def snhip_block_norm_backward(self, handle, desc, workspace, nbytes):
            return self.check(desc._obj.rows, workspace, nbytes)

    def run(number):
        w = Wrapper(number)

        def on(shape, type_="float32"):
            t = Stub(shape, type_)
            t.Wrapper = t._lib = w
            return t
        for k in range(60):
            rows = 3 + number + k
            e.BackwardPropagation(on((7, 6)), on((rows,), "int32"), on((rows, 6)))
            n.BackwardPropagation(on((rows, 6)), on((rows, 6)), on((rows, 6)), preStatistics=on((rows, 2)), dPreWeight=on((6,)))
    threads = [threading.Thread(target=run, args=(number,)) for number in (1, 2, 3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_clears_its_states_where_its_steps_go(bits):
    """Parameters of two wrappers of a device: the states are cleared by the one that the steps are issued by, and are clear
    before the plan is made."""
    from sharpnet_amd import optimizer
    log = []

    class Wrapper:
        device_id = 0

        def __init__(self, name):
            self.lib, self.handle, self.made = self, name, 0

        def allocate(self, nbytes):
            self.made += 1
            return A + (self.made << 20)

        def release(self, pointer, nbytes):
            pass

        def synchronize(self):
            log.append(("wait", self.handle))

        def snhip_memset32(self, handle, *args):
            log.append(("clear", handle))
            return 0

        def snhip_adamw_create(self, handle, *args):
            log.append(("create", handle))
            return 0
    first, second = Wrapper("first"), Wrapper("second")
    tensors = [Stub((300,)) for _ in range(4)]
    for t, w in zip(tensors, (first, second, first, second)):
        t.Wrapper = t._lib = w
    opt = optimizer.AdamW(tensors[:2], tensors[2:], stateBits=bits)
    clears = 2 * (2 if bits == 32 else 4)
    assert log == [("clear", "first")] * clears + [("wait", "first"), ("create", "first")]
    opt._plan = None  # (nothing to destroy)


def test_adamw_after_its_end():
    from sharpnet_amd import optimizer
    tensors = [Stub((3, 4)) for _ in range(4)]
    opt = optimizer.AdamW([], [])
    opt.Step()
    assert opt.StepCount == 1
    opt.Dispose()
    with pytest.raises(RuntimeError):
        opt.Step()
    assert opt.StepCount == 1
    opt = optimizer.AdamW.__new__(optimizer.AdamW)
    opt._disposed, opt._plan, opt._memory, opt.StepCount = False, None, tensors, 3
    tensors[2]._disposed = True
    with pytest.raises(RuntimeError):
        opt.Step()
    assert opt.StepCount == 3


# ---- the plain forms ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("pre,post,gate_rows,activation", [
    ("layer", "layer", 0, "sigmoid"), ("rms", "rms", 2, "tanh"), ("layer", None, 1, None), (None, "layer", 3, "sigmoid"),
    ("rms", "layer", None, None), ("layer", None, None, None)])
def test_plain_block_norm_gradients_against_differences(pre, post, gate_rows, activation):
    """Central differences in 64 bits with steps of 1e-5: off by the third derivative times 1e-10 and by rounding of
    1e-16 / 1e-5, both far below 1e-7."""
    rng = np.random.default_rng(0)
    rows, dim, eps, scale = 5, 7, 1e-3, np.float32(0.7)
    x = rng.normal(0, 1, (rows, dim))
    y = rng.normal(0, 1, (rows, dim)) if post or gate_rows is not None else None
    gate = None if gate_rows is None else rng.normal(0, 1, dim if gate_rows == 0 else (-(-rows // gate_rows), dim))
    weights = {}
    for which, kind in (("pre", pre), ("post", post)):
        if kind:
            weights[which + "_weight"], weights[which + "_bias"] = rng.normal(1, 0.3, dim), rng.normal(0, 0.3, dim)
    gu, gh = rng.normal(0, 1, (rows, dim)), rng.normal(0, 1, (rows, dim))

    def outputs():
        return ref.block_norm_forward(x, y, gate, gate_rows or 0, pre, post, weights, scale, eps, activation, "float32", "float32")

    def loss():
        o = outputs()
        return ((o["u"][0] * gu).sum() if "u" in o else 0.0) + ((o["h"][0] * gh).sum() if pre else 0.0)

    u = outputs()["u"][0] if y is not None else x
    stats = {}
    if pre:
        stats["pre"] = np.concatenate(ref.statistics(u, pre, eps), 1)
    if post:
        stats["post"] = np.concatenate(ref.statistics(y, post, eps), 1)
    got = ref.block_norm_backward(u, gh if pre else None, gu if y is not None else None, y, gate, gate_rows or 0, pre, post, weights, stats,
                                  scale, activation, "float32", "float32")
    inputs = {"dx": x, "dy": y, "d_gate": gate, **{"d_" + k: v for k, v in weights.items()}}
    for name, a in inputs.items():
        if a is None:
            continue
        flat, want = a.reshape(-1), got[name][0].reshape(-1)
        for i in range(flat.size):
            old = flat[i]
            flat[i] = old + 1e-5
            up = loss()
            flat[i] = old - 1e-5
            down = loss()
            flat[i] = old
            assert abs((up - down) / 2e-5 - want[i]) < 1e-7 * (1 + abs(want[i])), (name, i)


def test_plain_embedding_gradient_is_the_transpose_of_the_lookup():
    rng = np.random.default_rng(1)
    ids = np.array([3, -1, 0, 3, 9, 4, 3], np.int64)
    W, dy = rng.normal(0, 1, (5, 4)), rng.normal(0, 1, (7, 4))
    g, _ = ref.embedding_backward(ids, dy, 5, 0.5)
    assert abs((ref.embedding_forward(ids, W, 0.5) * dy).sum() - (g * W).sum()) < 1e-12
    assert np.array_equal(ref.valid_ids(np.array([0.9, -0.9, 4.99, 5.0, np.nan, -1.0, np.inf], np.float32), 5), [0, 0, 4, -1, -1, -1, -1])


def test_plain_8_bit_formats_are_torchs():
    import torch
    codes = torch.arange(256, dtype=torch.int32).to(torch.uint8)
    for table, type_ in ((ref.E4M3, torch.float8_e4m3fn), (ref.E5M2, torch.float8_e5m2)):
        want = codes.view(type_).float().numpy()
        assert np.array_equal(table, want, equal_nan=True)


def test_plain_random_words_are_the_published_ones():
    """The known answers that the generator's authors publish for philox4x32-10."""
    f = 0xFFFFFFFF
    for counter, key, want in (((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
                               ((f, f, f, f), (f, f), (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
                               ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
                                (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        assert tuple(int(x) for x in ref.philox(counter, key)) == want


def test_plain_8_bit_storage_rounds_to_a_neighbour_and_keeps_the_mean():
    rng = np.random.default_rng(2)
    x = (rng.normal(0, 1, 2048) * np.exp(rng.normal(0, 4, 2048))).astype(np.float32)
    x[:100] = 0
    for store, table, v in ((ref.store_m, ref.E4M3, x), (ref.store_v, ref.E5M2, np.abs(x))):
        draws = []
        for k in range(64):
            code, scale = store(v, ref.random_words(v.size, 0, k, 7))
            draws.append(ref.load8(code, scale, table).astype(np.float64))
        draws = np.array(draws)
        unit = np.repeat(ref.power(scale.astype(np.int64) - 127), 256).astype(np.float64)
        positive = np.unique(np.abs(table[np.isfinite(table)])).astype(np.float64)
        a = np.abs(v.astype(np.float64)) / unit
        below = positive[np.searchsorted(positive, a, side="right") - 1]
        above = positive[np.minimum(np.searchsorted(positive, a), positive.size - 1)]
        got = np.abs(draws) / unit
        lifted = (got == positive[1]) & (a > 0) & (a < positive[1])          # v: never zero
        assert np.all((got == below) | (got == above) | lifted)
        assert np.all(draws[:, v == 0] == 0)
        # the mean of 64 draws: a standard deviation of half a step / 8 at most; six of them
        normal = a >= positive[1]
        assert np.all(np.abs(got.mean(0) - a)[normal] <= (6 / 16 * (above - below) + 2.0 ** -16 * (above - below))[normal])
