"""What the layer norm, the activations kept in 8 bits and the loss over a vocabulary refuse, without a GPU: arguments are looked at
before anything is launched."""
import ctypes

import pytest
import torch

BF16 = torch.bfloat16


@pytest.fixture()
def p():
    buf = (ctypes.c_char * 8192)()
    yield (ctypes.cast(buf, ctypes.c_void_p).value + 255) & ~255


def c(name, *args):
    from hpfp8 import _lib
    lib = _lib.load()
    return getattr(lib, name)(*args), lib.hpfp8_last_error().decode()


def test_rows_in_8_bits(p):
    assert c("hpfp8_quantize_rows", p, 3, 4, 8, 8, p, p, None)[0] == -1
    assert c("hpfp8_quantize_rows", p, 0, -1, 8, 8, p, p, None)[0] == -2
    assert c("hpfp8_quantize_rows", p, 0, 4, 8, -8, p, p, None)[0] == -2
    assert c("hpfp8_quantize_rows", p + 1, 0, 4, 8, 8, p, p, None)[0] == -3
    assert c("hpfp8_quantize_rows", p + 2, 1, 4, 8, 8, p, p, None)[0] == -3
    assert c("hpfp8_quantize_rows", p, 0, 4, 8, 8, p, None, None)[0] == -1
    assert c("hpfp8_quantize_rows", p, 0, 1, 1 << 40, 8, p, p, None)[0] == -2
    assert c("hpfp8_quantize_rows", None, 0, 0, 8, 8, None, None, None)[0] == 0
    assert c("hpfp8_quantize_rows", None, 0, 8, 0, 0, None, None, None)[0] == 0
    assert c("hpfp8_dequantize_rows", p, p, 4, 8, p, 7, None)[0] == -1
    assert c("hpfp8_dequantize_rows", p, p, 4, 8, p + 1, 2, None)[0] == -3
    assert c("hpfp8_dequantize_rows", None, p, 4, 8, p, 2, None)[0] == -1
    assert c("hpfp8_dequantize_rows", None, None, 0, 8, None, 2, None)[0] == 0


def test_activations(p):
    assert c("hpfp8_activation_forward", p, 0, 4, 8, 8, 4, p, None, None, None)[0] == -1
    assert c("hpfp8_activation_forward", p, 0, 4, 8, 8, 0, p, p, None, None)[0] == -1          # codes without scales
    assert c("hpfp8_activation_forward", p, 0, 4, 8, 8, 0, p + 1, None, None, None)[0] == -3
    assert c("hpfp8_activation_forward", None, 0, 0, 8, 8, 0, None, None, None, None)[0] == 0
    assert c("hpfp8_activation_backward", p, p, 8, p, p, 0, 4, 8, 0, p, None)[0] == -1         # both x and its codes
    assert c("hpfp8_activation_backward", p, None, 8, None, None, 0, 4, 8, 0, p, None)[0] == -1
    assert c("hpfp8_activation_backward", None, None, 8, None, None, 0, 4, 0, 0, None, None)[0] == 0


def test_layer_norm(p):
    f, b = "hpfp8_layer_norm_forward", "hpfp8_layer_norm_backward"
    assert c(f, p, 0, 4, 16385, 16385, None, None, 0, 1e-5, p, None, None, None, None, None)[0] == -2
    assert c(f, p, 0, 4, 0, 0, None, None, 0, 1e-5, p, None, None, None, None, None)[0] == -2
    assert c(f, p, 5, 4, 8, 8, None, None, 0, 1e-5, p, None, None, None, None, None)[0] == -1
    assert c(f, p, 0, 4, 8, 8, None, None, 0, 1e-5, p, None, None, p, None, None)[0] == -1
    assert c(f, p, 0, 4, 8, 8, p + 2, None, 1, 1e-5, p, None, None, None, None, None)[0] == -3
    assert c(f, None, 0, 0, 8, 8, None, None, 0, 1e-5, None, None, None, None, None, None)[0] == 0
    assert c(b, p, 8, p, 8, None, None, None, p, 0, 4, 8, None, 0, p, p, p, p, None)[0] == -1  # x without its mean
    assert c(b, p, 8, None, 8, p, None, None, p, 0, 4, 8, None, 0, p, p, p, p, None)[0] == -1
    assert c(b, p, 8, p, 8, p, None, None, p, 0, 4, 8, None, 0, p, p, p, None, None)[0] == -1  # no workspace
    assert c("hpfp8_layer_norm_partials", 0, 8)[0] == 0 and c("hpfp8_layer_norm_partials", 1, 16385)[0] == 0
    assert c("hpfp8_layer_norm_partials", 1, 7168)[0] == 1 and c("hpfp8_layer_norm_partials", 1 << 20, 7168)[0] == 256


def test_linear_cross_entropy(p):
    f, piece = "hpfp8_linear_cross_entropy_forward", "hpfp8_linear_cross_entropy_piece"

    def forward(x=p, ld_x=64, w=p, ld_w=64, target=p, tokens=4, hidden=64, vocab=10, smoothing=0.0, reduction=0, stats=p, sums=None, out=None):
        return c(f, x, ld_x, w, ld_w, target, tokens, hidden, vocab, -100, smoothing, reduction, stats, sums, p, None, p, out, out, None)[0]
    assert forward(hidden=63) == -2 and forward(ld_x=60) == -2 and forward(ld_w=56) == -2 and forward(vocab=0) == -2
    assert forward(vocab=(1 << 24) + 1) == -2 and forward(tokens=(1 << 22) + 1) == -2 and forward(tokens=-1) == -2
    assert forward(ld_x=1 << 21) == -2
    assert forward(reduction=3) == -1 and forward(reduction=1) == -1 and forward(smoothing=1.5) == -1 and forward(smoothing=0.1) == -1
    assert forward(x=p + 2) == -3 and forward(stats=None) == -1 and forward(target=None) == -1
    assert forward(tokens=0, x=None, target=None) == 0

    def backward(first=0, width=10, dx=None, dw=None, x_t=None, dw_type=0, dw_add=0, dl=p, tokens=4, splits=1):
        return c(piece, p, 64, x_t, p, 64, p, tokens, 64, 10, first, width, -100, 0.0, p, p, 0, None, dl, p, dx, splits, 0, dw, dw_type, dw_add, None)[0]
    assert backward(first=5, width=6) == -2 and backward(width=0) == -2 and backward(first=-1) == -2
    assert backward(dw=p) == -1 and backward(dw_type=2) == -1 and backward(dw_add=1) == -1 and backward(dl=None) == -1
    assert backward(dl=p + 8) == -3 and backward(dx=p, splits=0) == -1 and backward(dx=p, splits=33) == -1 and backward(dx=p, splits=2) == -1
    assert backward(tokens=0) == 0
    t = "hpfp8_linear_cross_entropy_rows_t"
    assert c(t, p, 10, 64, 64, None, 0, p, 56, None)[0] == -2 and c(t, p, 10, 60, 64, None, 0, p, 64, None)[0] == -2
    assert c(t, None, 10, 64, 64, None, 0, p, 64, None)[0] == -1 and c(t, None, 0, 64, 64, None, 0, None, 0, None)[0] == 0
    assert c("hpfp8_linear_cross_entropy_round", p, 12, 1, p, None)[0] == -2 and c("hpfp8_linear_cross_entropy_round", p, 16, 1, None, None)[0] == -1
    assert c("hpfp8_linear_cross_entropy_round", p, 16, 0, p, None)[0] == -1
    assert c("hpfp8_linear_cross_entropy_reduce", p, p, 4, -100, 0, p, p, None)[0] == -1
    assert c("hpfp8_linear_cross_entropy_reduce", p, p, 4, -100, 1, p, None, None)[0] == -1


def test_tensors_that_are_not_on_the_gpu_and_wrong_arguments():
    import hpfp8
    x, w, t = torch.zeros(4, 64, dtype=BF16), torch.zeros(10, 64, dtype=BF16), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: hpfp8.layer_norm(x, 64), lambda: hpfp8.activation(x, "silu"), lambda: hpfp8.quantize_activation(x),
                 lambda: hpfp8.linear_cross_entropy(x, w, t)):
        with pytest.raises(ValueError, match="must live on the GPU"):
            call()
    with pytest.raises(ValueError, match="kind must be one of"):
        hpfp8.activation(x, "relu")
    with pytest.raises(ValueError, match="reduction must be one of"):
        hpfp8.linear_cross_entropy(x, w, t, reduction="max")
    with pytest.raises(ValueError, match="label_smoothing"):
        hpfp8.linear_cross_entropy(x, w, t, label_smoothing=-0.1)
    for call in (lambda: hpfp8.layer_norm(x.double(), 64), lambda: hpfp8.activation(x.int(), "gelu"), lambda: hpfp8.quantize_activation(x.double())):
        with pytest.raises(TypeError, match="bfloat16, float16 or float32"):
            call()
    with pytest.raises(TypeError, match="must be a torch.Tensor"):
        hpfp8.quantize_activation([1.0])
    with pytest.raises(TypeError, match="dtypes"):
        with hpfp8.keep_activations_8bit(dtypes=(torch.float64,)):
            pass
    with hpfp8.keep_activations_8bit(min_elements=1):                 # (tensors that are not on the GPU stay as they are)
        y = torch.ones(4, requires_grad=True) * 3
        (y * y).sum().backward()


class Recorder(torch.Tensor):
    calls = []

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        Recorder.calls.append((func, len(args), dict(kwargs or {})))
        return "handed off"


def test_subclasses_are_handed_the_call():
    import hpfp8
    x = torch.zeros(4, 64).as_subclass(Recorder)
    Recorder.calls.clear()
    assert hpfp8.layer_norm(x, 64, keep_8bit=True) == "handed off"
    assert hpfp8.activation(x, "silu") == "handed off"
    assert hpfp8.linear_cross_entropy(x, torch.zeros(3, 64), torch.zeros(4), reduction="sum") == "handed off"
    assert [f.__name__ for f, _, _ in Recorder.calls] == ["layer_norm", "activation", "linear_cross_entropy"]
    assert [k for _, _, k in Recorder.calls] == [{"keep_8bit": True}, {}, {"reduction": "sum"}]


def test_sizes_that_31_bits_do_not_address(p):
    """256 rows of a workspace that has a column for each token, or for each of a piece's, span less than 2 GiB."""
    def forward(tokens):
        return c("hpfp8_linear_cross_entropy_forward", None, 8, p, 8, p, tokens, 8, 10, -100, 0.0, 0, p, None, p, None, p, None, None, None)[0]
    assert forward((1 << 21) + 1) == -2 and forward(1 << 21) == -1           # (the second for its null x)

    def piece(width):
        return c("hpfp8_linear_cross_entropy_piece", None, 8, None, p, 8, p, 4, 8, 1 << 24, 0, width, -100, 0.0, p, p, 0, None, p, p, None, 1, 0, None,
                 0, 0, None)[0]
    assert piece((1 << 21) + 1) == -2 and piece(1 << 21) == -1


def test_codes_and_scales_of_other_types():
    from hpfp8.kept import Fp8Activation
    codes, scale_inv = torch.zeros(4, 64, dtype=torch.float8_e4m3fn), torch.ones(4, 1)
    for wrong in ((codes.float(), scale_inv), (codes, scale_inv.double())):
        with pytest.raises(TypeError):
            Fp8Activation(*wrong, BF16).dequantize()
    with pytest.raises(ValueError, match="must live on the GPU"):
        Fp8Activation(codes, scale_inv, BF16).dequantize()


def test_parts_of_the_forward():
    from hpfp8 import _lib
    parts = _lib.load().hpfp8_cross_entropy_parts
    assert parts(0, 64, 100) == 0 and parts(4, 64, 0) == 0
    assert parts(4, 64, 100) == 2 and parts(4096, 7168, 131072) == 512
    for tokens in (1, 64, 65, 300, 5000):
        for vocab in (1, 64, 257, 5000, 131072):
            assert parts(tokens, 512, vocab) in [-(-vocab // cols) for cols in (64, 128, 256)]


@pytest.mark.parametrize("wrong", ["device", "start", "shape", "type", "strides"])
def test_a_main_grad_that_the_kernels_cannot_add_onto(wrong, monkeypatch):
    """Refused by the call, and by the backward if it was put there in between: before anything is launched."""
    import hpfp8
    from hpfp8 import _lib, loss, ops
    launched = []
    monkeypatch.setattr(_lib, "call", lambda name, *args: launched.append(name))
    monkeypatch.setattr(ops, "_check_device", lambda *args: None)
    monkeypatch.setattr(ops, "_stream", lambda: None)
    w = torch.nn.Parameter(torch.zeros(10, 64, dtype=BF16))
    w.main_grad = {"device": torch.zeros(10, 64, device="meta"), "start": torch.zeros(643)[3:].view(10, 64), "shape": torch.zeros(64, 10),
                   "type": torch.zeros(10, 64, dtype=BF16), "strides": torch.zeros(64, 10).t()}[wrong]
    x, t = torch.zeros(4, 64, dtype=BF16, requires_grad=True), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="main_grad"):
        hpfp8.linear_cross_entropy(x, w, t, apply_grad_on_fp32_main_grad=True)
    with pytest.raises(ValueError, match="main_grad"):
        loss._backward(torch.ones(()), x.detach(), w.detach(), t, torch.zeros(4), torch.ones(()), -100, 1, 0.0, True, True, w)
    assert not launched


def test_saved_tensors_that_a_hook_handed_back_as_something_else(monkeypatch):
    """Left on the CPU, shortened or of another type: refused before anything is launched."""
    from hpfp8 import _lib, kept, loss, norm, ops
    launched = []
    monkeypatch.setattr(_lib, "call", lambda name, *args: launched.append(name))
    monkeypatch.setattr(ops, "_stream", lambda: None)
    x, go, codes, one = torch.zeros(4, 64, dtype=BF16), torch.zeros(4, 64, dtype=BF16), torch.zeros(4, 64, dtype=torch.float8_e4m3fn), torch.zeros(4, 1)
    t, row = torch.zeros(4, dtype=torch.int64), torch.zeros(4)
    code = kept._TYPES[BF16]
    calls = {kept._backward: [(go, x, None, False, 0, x.shape), (go, codes, one, True, 0, x.shape)],
             norm._backward: [(go, x, row, row, x[0], False, 64, x.shape, code, (64,), code, True, True),
                              (go, codes, one, row, x[0], True, 64, x.shape, code, (64,), code, True, True)],
             loss._backward: [(torch.ones(()), x, x, t, row, torch.ones(()), -100, 1, 0.0, True, True)]}
    for function, each in calls.items():
        for args in each:
            with pytest.raises(ValueError, match="must live on the GPU"):
                function(*args)
    monkeypatch.setattr(ops, "_check_device", lambda *args: None)
    for function, each in calls.items():
        for args in each:
            saved = [i for i, a in enumerate(args) if i > 0 and isinstance(a, torch.Tensor)]
            for i in saved:
                wrongs = [args[i].to(torch.float64)]
                if not (function is loss._backward and i == 2):              # (the vocabulary is the weight's own)
                    wrongs.append(args[i][:-1] if args[i].dim() else args[i].expand(2))
                for wrong in wrongs:
                    with pytest.raises(ValueError, match="came back as"):
                        function(*args[:i], wrong, *args[i + 1:])
    assert not launched


def test_rows_that_start_between_two_vectors_or_have_odd_strides_are_copied():
    """Contiguous tensors among them: views in a flat buffer, a single row cut out of columns."""
    from hpfp8.loss import _rows
    flat = torch.arange(1 + 5 * 64).to(BF16)
    for x in (flat[1:].view(5, 64), flat[1:65].view(1, 64), flat[:64].view(64, 1).t(), flat[:320].view(64, 5).t(), flat[:64].expand(5, 64),
              flat[:63 * 5].view(5, 63)[:, 3:59]):
        rows = _rows(x)
        assert torch.equal(rows, x) and rows.data_ptr() % 16 == 0 and rows.stride(1) == 1 and rows.stride(0) % 8 == 0 and rows.stride(0) >= rows.shape[1]
    assert _rows(flat[:320].view(5, 64)).data_ptr() == flat.data_ptr()


def test_saved_rows_in_8_bits(p):
    q, d = "hpfp8_quantize_saved_rows", "hpfp8_dequantize_saved_rows"
    assert c(q, p, 3, 4, 8, 8, p, p, None)[0] == -1 and c(q, p, 0, -1, 8, 8, p, p, None)[0] == -2 and c(q, p + 1, 0, 4, 8, 8, p, p, None)[0] == -3
    assert c(q, p, 0, 4, 8, 8, p, None, None)[0] == -1 and c(q, p, 0, 1, 1 << 40, 8, p, p, None)[0] == -2 and c(q, None, 0, 0, 8, 8, None, None, None)[0] == 0
    assert c(d, p, p, 4, 8, p, 7, None)[0] == -1 and c(d, p, p, 4, 8, p + 1, 2, None)[0] == -3 and c(d, None, p, 4, 8, p, 2, None)[0] == -1
    assert c(d, None, None, 0, 8, None, 2, None)[0] == 0


def test_a_weight_gradient_of_no_tokens_is_checked_too(p):
    def piece(dw, dw_add=0, dw_type=0):
        return c("hpfp8_linear_cross_entropy_piece", None, 64, None, None, 64, None, 0, 64, 10, 0, 10, -100, 0.0, None, None, 0, None, None, None, None, 1, 0,
                 dw, dw_type, dw_add, None)[0]
    assert piece(p + 8) == -3 and piece(p, 1, 1) == 0 and piece(None) == 0
