"""CPU-only checks of the image-token attention entry points: what they refuse, before anything reaches a GPU, and the
oracle's own formulas against an independent statement of them."""
import ctypes

import numpy as np
import pytest

import image_attention_ref as ref
from conftest import load_package

A = 1 << 20  # an aligned address that no refused call may follow


@pytest.fixture(scope="module")
def mbx():
    return load_package()


@pytest.fixture(scope="module")
def blank():
    """Memory of a context's size that the argument checks come before: none of them looks into it."""
    return ctypes.create_string_buffer(4096)


def _refused(mbx, status, text):
    message = mbx.abi.lib().mbx_last_error().decode()
    assert status == mbx.abi.ERR_INVALID_ARGUMENT, message
    assert text in message, message


ROPE = dict(x=A, x_dtype=0, n=2, tokens=6, x_stride=24 * 4, heads=2, kv_heads=1, dim=24, norm=1, q_gamma=None,
            k_gamma=None, eps=1e-6, positions=A, position_items=1, axis_dims=(0, 8, 8), theta=1e4, pairing=0, q=A,
            k=A, v=A, out_dtype=0)


@pytest.mark.parametrize("change,text", [
    (dict(n=-1), "shape"), (dict(tokens=-1), "shape"), (dict(tokens=1 << 40), "shape"),
    (dict(heads=0, kv_heads=0), "head"), (dict(heads=-1), "head"), (dict(dim=20), "dim"), (dict(dim=0), "dim"),
    (dict(dim=264, x_stride=2112), "dim"), (dict(x_dtype=3), "dtype"), (dict(out_dtype=-1), "dtype"),
    (dict(x_dtype=1, out_dtype=0), "type"), (dict(x_dtype=1, out_dtype=2), "type"), (dict(pairing=2), "pairing"),
    (dict(x_stride=95), "stride"), (dict(x_stride=98), "16 bytes"), (dict(x=A + 4), "aligned"),
    (dict(q=A + 8), "aligned"), (dict(q=None), "q"), (dict(k=None), "k"), (dict(v=A + 2), "aligned"),
    (dict(x=None), "x"), (dict(axis_dims=None), "axis_dims"), (dict(axis_dims=(0, 9, 8)), "axis_dims"),
    (dict(axis_dims=(8, 8, 10)), "exceed"), (dict(axis_dims=(0, -8, 8)), "axis_dims"), (dict(theta=0.0), "theta"),
    (dict(theta=float("nan")), "theta"), (dict(position_items=3), "position_items"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("inf")), "eps")])
def test_qkv_norm_rope_refuses(mbx, blank, change, text):
    a = {**ROPE, **change}
    dims = None if a["axis_dims"] is None else (ctypes.c_int64 * 3)(*a["axis_dims"])
    _refused(mbx, mbx.abi.lib().mbx_qkv_norm_rope(
        blank, a["x"], a["x_dtype"], a["n"], a["tokens"], a["x_stride"], a["heads"], a["kv_heads"], a["dim"],
        a["norm"], a["q_gamma"], a["k_gamma"], a["eps"], a["positions"], a["position_items"], dims, a["theta"],
        a["pairing"], a["q"], a["k"], a["v"], a["out_dtype"]), text)


BLOCK = dict(q=A, q_stride=64, k=A, k_stride=32, v=A, v_stride=32, dtype=1, n=2, nq=130, nk=70, heads=2, kv_heads=1,
             dim=32, block_k=64, topk=2, scale=1.0, index=A, out=A, workspace=A, workspace_bytes=1 << 30)
BAD_BLOCKS = [
    (dict(n=-1), "shape"), (dict(nq=-1), "shape"), (dict(nk=1 << 31), "shape"), (dict(heads=3, kv_heads=2), "kv_heads"),
    (dict(heads=0), "kv_heads"), (dict(kv_heads=0), "kv_heads"), (dict(n=40000), "65535"), (dict(dim=36), "dim"),
    (dict(dim=0), "dim"), (dict(block_k=48), "block_k"), (dict(block_k=256), "block_k"), (dict(topk=-1), "topk"),
    (dict(topk=1 << 20), "topk")]
BAD_TENSORS = [
    (dict(dtype=3), "dtype"), (dict(q_stride=63), "stride"), (dict(k_stride=31), "stride"),
    (dict(q_stride=68), "16 bytes"), (dict(q=A + 2), "aligned"), (dict(k=A + 8), "aligned"), (dict(q=None), "q"),
    (dict(k=None), "k"), (dict(index=None), "index"), (dict(workspace=None), "workspace"),
    (dict(workspace=A + 16), "workspace"), (dict(workspace_bytes=0), "workspace")]


def _select(mbx, blank, a):
    return mbx.abi.lib().mbx_block_select(blank, a["q"], a["q_stride"], a["k"], a["k_stride"], a["dtype"], a["n"],
                                          a["nq"], a["nk"], a["heads"], a["kv_heads"], a["dim"], a["block_k"], None,
                                          a["topk"], a["index"], a["workspace"], a["workspace_bytes"])


def _attend(mbx, blank, a):
    return mbx.abi.lib().mbx_block_attention(blank, a["q"], a["q_stride"], a["k"], a["k_stride"], a["v"],
                                             a["v_stride"], a["dtype"], a["n"], a["nq"], a["nk"], a["heads"],
                                             a["kv_heads"], a["dim"], a["block_k"], None, a["index"], a["topk"],
                                             a["scale"], a["out"], a["workspace"], a["workspace_bytes"])


@pytest.mark.parametrize("change,text", BAD_BLOCKS + BAD_TENSORS + [(dict(dim=264, q_stride=528, k_stride=264), "dim")])
def test_block_select_refuses(mbx, blank, change, text):
    _refused(mbx, _select(mbx, blank, {**BLOCK, **change}), text)


@pytest.mark.parametrize("change,text", BAD_BLOCKS + [c for c in BAD_TENSORS if "workspace" not in c[1]] + [
    (dict(dim=136, q_stride=272, k_stride=136, v_stride=136), "dim"), (dict(v_stride=24), "stride"),
    (dict(v=A + 4), "aligned"), (dict(v=None), "v"), (dict(out=None), "out"), (dict(out=A + 8), "aligned"),
    (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale")])
def test_block_attention_refuses(mbx, blank, change, text):
    _refused(mbx, _attend(mbx, blank, {**BLOCK, **change}), text)


def test_block_attention_refuses_a_small_workspace(mbx, blank):
    need = ctypes.c_size_t()
    a = {**BLOCK, "nq": 1, "nk": 1 << 20, "topk": 512, "n": 1, "dtype": 0}
    assert mbx.abi.lib().mbx_block_attention_workspace(a["dtype"], a["n"], a["nq"], a["nk"], a["heads"],
                                                       a["kv_heads"], a["dim"], a["block_k"], a["topk"],
                                                       ctypes.byref(need)) == mbx.abi.OK
    assert need.value > 0
    _refused(mbx, _attend(mbx, blank, {**a, "workspace_bytes": need.value - 1}), "workspace")
    _refused(mbx, _attend(mbx, blank, {**a, "workspace": None}), "workspace")


@pytest.mark.parametrize("change,text", BAD_BLOCKS[:-2])
def test_workspace_sizes_refuse_what_the_calls_refuse(mbx, change, text):
    a, need, lib = {**BLOCK, **change}, ctypes.c_size_t(), mbx.abi.lib()
    shape = [a[s] for s in ("n", "nq", "nk", "heads", "kv_heads", "dim", "block_k")]
    _refused(mbx, lib.mbx_block_select_workspace(*shape, ctypes.byref(need)), text)
    _refused(mbx, lib.mbx_block_attention_workspace(a["dtype"], *shape, a["topk"], ctypes.byref(need)), text)
    _refused(mbx, lib.mbx_block_select_workspace(*[BLOCK[s] for s in ("n", "nq", "nk", "heads", "kv_heads", "dim",
                                                                      "block_k")], None), "bytes")


@pytest.mark.parametrize("change", [dict(nq=1 << 30, heads=1024, nk=1 << 30),  # a size that would wrap around
                                    dict(nq=64 * 65535 * 128 + 1, n=1, heads=1)])
def test_block_select_refuses_too_many_query_blocks(mbx, blank, change):
    a, need = {**BLOCK, **change}, ctypes.c_size_t()
    a.update(q_stride=a["heads"] * a["dim"])
    shape = [a[s] for s in ("n", "nq", "nk", "heads", "kv_heads", "dim", "block_k")]
    _refused(mbx, mbx.abi.lib().mbx_block_select_workspace(*shape, ctypes.byref(need)), "query blocks")
    _refused(mbx, _select(mbx, blank, a), "query blocks")


def test_null_context(mbx):
    _refused(mbx, _select(mbx, None, BLOCK), "context")
    _refused(mbx, _attend(mbx, None, BLOCK), "context")


def test_nothing_to_do_is_no_error(mbx, blank):
    """Empty work returns before the device: no query, no item, nothing to choose."""
    for change in (dict(n=0), dict(nq=0), dict(topk=0)):
        assert _select(mbx, blank, {**BLOCK, **change}) == mbx.abi.OK
    for change in (dict(n=0), dict(nq=0)):
        assert _attend(mbx, blank, {**BLOCK, **change}) == mbx.abi.OK


def test_python_front_end_refuses_mismatched_tensors(mbx):
    def t(shape, dtype=np.float16):
        return mbx.DeviceTensor.wrap(None, A, shape, dtype=dtype)
    q, k = t((1, 4, 2, 16)), t((1, 5, 1, 16))
    index = t((1, 2, 1, 3), np.int32)
    with pytest.raises(ValueError, match="index"):
        mbx.block_attention(q, k, k, t((1, 2, 2, 3), np.int32), workspace=q, out=q)
    with pytest.raises(ValueError, match="index"):
        mbx.block_attention(q, k, k, t((1, 2, 1, 3), np.float32), workspace=q, out=q)
    with pytest.raises(ValueError, match="v must"):
        mbx.block_attention(q, k, t((1, 6, 1, 16)), index, workspace=q, out=q)
    with pytest.raises(ValueError, match="key_mask"):
        mbx.block_attention(q, k, k, index, key_mask=t((1, 4), np.uint8), workspace=q, out=q)
    with pytest.raises(ValueError, match="type"):
        mbx.block_select(q, t((1, 5, 1, 16), np.float32), 3, workspace=q, out=index)
    with pytest.raises(ValueError, match="out"):
        mbx.block_select(q, k, 2, workspace=q, out=index)
    x = t((1, 4, 4 * 16), np.float32)
    with pytest.raises(ValueError, match="q must"):
        mbx.qkv_norm_rope(x, 2, 1, 16, out=(t((1, 4, 1, 16)), t((1, 4, 1, 16)), t((1, 4, 1, 16))))
    with pytest.raises(ValueError, match="positions"):
        mbx.qkv_norm_rope(x, 2, 1, 16, positions=t((1, 5, 3), np.float32),
                          out=(t((1, 4, 2, 16)), t((1, 4, 1, 16)), t((1, 4, 1, 16))))


def test_python_front_end_refuses_tensors_of_another_device(mbx):
    class Device:  # a context, as far as the checks look into it
        def __init__(self, device):
            self.device, self.handle = device, None
    here, same, other = Device(0), Device(0), Device(1)

    def t(ctx, shape, dtype=np.float16):
        return mbx.DeviceTensor.wrap(ctx, A, shape, dtype=dtype)
    shapes = dict(q=(1, 4, 2, 16), k=(1, 5, 1, 16), v=(1, 5, 1, 16), index=(1, 2, 1, 3), key_mask=(1, 5),
                  workspace=(8,), out=(1, 4, 2, 16))
    kinds = dict(index=np.int32, key_mask=np.uint8, workspace=np.uint8)

    def attend(**at):
        a = {s: t(at.get(s, here), shape, kinds.get(s, np.float16)) for s, shape in shapes.items()}
        return mbx.block_attention(a.pop("q"), a.pop("k"), a.pop("v"), a.pop("index"), **a)

    def select(**at):
        a = {s: t(at.get(s, here), shapes[s], kinds.get(s, np.float16)) for s in ("q", "k", "key_mask", "workspace")}
        return mbx.block_select(a.pop("q"), a.pop("k"), 3, out=t(at.get("out", here), shapes["index"], np.int32), **a)

    def rope(**at):
        parts = tuple(t(at.get(s, here), (1, 4, h, 16)) for s, h in (("q", 2), ("k", 1), ("v", 1)))
        return mbx.qkv_norm_rope(t(here, (1, 4, 64)), 2, 1, 16, positions=t(at.get("positions", here), (4, 3), np.float32),
                                 q_gamma=t(at.get("q_gamma", here), (16,), np.float32), out=parts)
    for call, names in ((attend, shapes), (select, ("q", "k", "key_mask", "workspace", "out")),
                        (rope, ("q", "k", "v", "positions", "q_gamma"))):
        for name in names:
            with pytest.raises(ValueError, match="device"):
                call(**{name: other})
            with pytest.raises(mbx.MbxError, match="context"):  # past the front end: there is no handle
                call(**{name: same})


def test_block_attention_refuses_other_results(mbx, blank):
    """The result is float32 or of the operands' type."""
    for dtype in (3 | mbx.abi.OUT_F32, 1 | 32, -1):
        _refused(mbx, _attend(mbx, blank, {**BLOCK, "dtype": dtype}), "dtype")

    def t(shape, dtype=np.float16):
        return mbx.DeviceTensor.wrap(None, A, shape, dtype=dtype)
    q, k, index = t((1, 4, 2, 16)), t((1, 5, 1, 16)), t((1, 2, 1, 3), np.int32)
    for out in (t((1, 4, 2, 16), mbx.bfloat16), t((1, 4, 2, 8), np.float32), t((1, 4, 2, 8))):
        with pytest.raises(ValueError, match="out"):
            mbx.block_attention(q, k, k, index, workspace=q, out=out)


def test_tensor_size_is_a_plain_integer(mbx):
    """A shape of NumPy's narrow integers must not wrap around (or warn) on its way to a size in bytes."""
    t = mbx.DeviceTensor(None, (np.int32(1 << 16), np.int32(1 << 16), np.uint8(3)), ptr=A)
    assert t.size == 3 << 32 and t.nbytes == 12 << 32 and type(t.size) is int and type(t.nbytes) is int
    assert mbx.DeviceTensor(None, (), ptr=A).size == 1 and mbx.DeviceTensor(None, (0, 5), ptr=A).size == 0


def test_float32_operators_refuse_the_16_bit_tensors(mbx):
    """The other operators work on float32: half-precision heads handed to one would be read past their end."""
    def t(shape, dtype=np.float32):
        return mbx.DeviceTensor.wrap(None, A, shape, dtype=dtype)

    class Weight:  # of a convolution; the checks come before its handle
        c_out, taps, handle = 16, 1, None
    image, vector, rows = (1, 4, 4, 16), (16,), (16, 16)
    calls = {
        "silu_inplace": [image], "add_inplace": [image, image], "bias_temb_add": [image, vector],
        "concat_channels": [image, image], "group_norm_apply": [image, (1, 16), (1, 16)],
        "layer_norm": [image, vector, vector], "depthwise3x3": [image, (16, 9), vector], "matmul": [rows, rows]}
    for dtype in (np.float16, mbx.bfloat16):
        for name, shapes in calls.items():
            for bad in range(len(shapes)):
                args = [t(s, dtype if i == bad else np.float32) for i, s in enumerate(shapes)]
                with pytest.raises(ValueError, match="float32"):
                    getattr(mbx, name)(*args, *([1e-5] if name == "layer_norm" else []))
        x, v, f = t(image, dtype), t(vector, dtype), t(vector)
        for call in (lambda: mbx.conv1x1(x, Weight), lambda: mbx.conv1x1(t(image), Weight, residual=x),
                     lambda: mbx.conv1x1(t(image), Weight, out=x), lambda: mbx.conv3x3(x, Weight),
                     lambda: mbx.conv3x3(t(image), Weight, bias=v),
                     lambda: mbx.conv3x3(t(image), Weight, prologue=(f, v, True)),
                     lambda: mbx.group_norm(x, 4, 1e-5, f, f), lambda: mbx.group_norm_affine(t(image), 4, 1e-5, v, f),
                     lambda: mbx.conv_group_norm_affine(x, Weight, 4, 1e-5, f, f)):
            with pytest.raises(ValueError, match="float32"):
                call()


def test_oracle_rotation_is_a_rotation():
    """Pairs keep their length, and a shift of all positions leaves products of equal shifts alone."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((1, 5, 2, 16))
    pos = rng.integers(0, 50, (1, 5, 3)).astype(np.float64)
    for halves in (False, True):
        y, size = ref.norm_rope(x, None, 0.0, False, pos, (4, 6, 4), 100.0, halves)
        z, _ = ref.norm_rope(x, None, 0.0, False, pos + 7, (4, 6, 4), 100.0, halves)
        assert np.allclose((y * y).sum(-1), (x * x).sum(-1))
        assert np.allclose(np.einsum("bthd,bshd->bhts", y, y), np.einsum("bthd,bshd->bhts", z, z))
        assert np.allclose(y[..., 14:], x[..., 14:]) and np.all(size >= np.abs(y) - 1e-12)


def test_oracle_attention_over_every_block_is_dense_attention():
    rng = np.random.default_rng(1)
    q, k, v = (rng.standard_normal((1, t, 2, 8)) for t in (150, 50, 50))
    index = np.broadcast_to(np.arange(4, dtype=np.int32), (1, 2, 2, 4))
    got, tol = ref.attention(q, k, v, index, 16, None, 0.3, "f32")
    s = np.einsum("bthd,bshd->bhts", q, k) * 0.3
    p = np.exp(s) / np.exp(s).sum(-1, keepdims=True)
    assert np.allclose(got, np.einsum("bhts,bshd->bthd", p, v)) and np.all(tol > 0)


def test_narrow_rounds_to_nearest():
    v = np.float32([1.0, 1.0 + 2 ** -8, 1.0 + 3 * 2 ** -8, -3.14159, 1e38, 0.0, np.inf, -np.inf, np.nan])
    got = ref.wide(ref.narrow(v, "bf16"))
    assert got[1] == 1.0 and got[2] == 1.0 + 2 ** -6 and np.isinf(got[6]) and np.isnan(got[8])
    ok = np.isfinite(v)
    assert np.all(np.abs(got[ok] - v[ok]) <= 2.0 ** -8 * np.abs(v[ok]))
