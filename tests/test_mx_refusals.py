"""What the microscaled operators and the scored routing refuse, and the oracle they are tested against (CPU only)."""

import pytest
import torch

import quantaweave_amd as qa
from quantaweave_amd import _lib
from quantaweave_amd.routing import check_rule
from tests import mx_oracle as ref


def test_cpu_tensors_are_refused():
    x = torch.randn(4, 64)
    codes, scales = ref.stored(torch.Generator().manual_seed(0), 8, 64)
    for call in (lambda: qa.mx_quantize(x), lambda: qa.mx_dequantize(codes, scales, 64),
                 lambda: qa.mx_matmul(x, codes, scales), lambda: qa.route_experts(x, 2),
                 lambda: qa.mx_grouped_swiglu(x, (codes, scales), (codes, scales), (codes, scales), torch.zeros(2).int())):
        with pytest.raises(RuntimeError, match="ROCm"):
            call()


@pytest.mark.parametrize("change,match", [
    (dict(score="tanh"), "score"), (dict(group_score="sum"), "group_score"), (dict(experts=0), "experts"),
    (dict(experts=1025), "experts"), (dict(groups=0), "groups"), (dict(groups=5), "groups"),
    (dict(top_groups=9), "top_groups"), (dict(top_k=0), "top_k"), (dict(top_k=33), "top_k"),
    (dict(experts=256, groups=1, top_groups=1, top_k=65), "top_k"), (dict(scale=float("nan")), "scale")])
def test_rules_that_no_kernel_takes(change, match):
    rule = dict(experts=64, top_k=8, score="sigmoid", groups=8, top_groups=4, group_score="top2", scale=1.0)
    check_rule(**rule)
    with pytest.raises(ValueError, match=match):
        check_rule(**{**rule, **change})


def test_entry_points_check_their_arguments_before_any_launch():
    lib = _lib.load()
    one = 64  # an address that is never read: the calls below are refused before a launch

    def refused(status, word):
        assert status == _lib.QW_ERR_INVALID and word in lib.qw_last_error(), lib.qw_last_error()

    route = lib.qw_moe_route_scored_from_logits
    refused(route(one, 4, 64, 65, 0, None, 1, 1, 2, 1, 1.0, one, one, one, None), b"top_k")
    refused(route(one, 4, 64, 2, 2, None, 1, 1, 2, 1, 1.0, one, one, one, None), b"score")
    refused(route(one, 4, 64, 2, 0, None, 7, 1, 2, 1, 1.0, one, one, one, None), b"groups")
    refused(route(one, 4, 64, 2, 0, None, 8, 9, 2, 1, 1.0, one, one, one, None), b"top_groups")
    refused(route(one, 4, 64, 9, 0, None, 8, 1, 2, 1, 1.0, one, one, one, None), b"top_k")
    refused(route(one, 4, 64, 2, 0, None, 8, 1, 3, 1, 1.0, one, one, one, None), b"group_top")
    refused(route(None, 4, 64, 2, 0, None, 8, 1, 2, 1, 1.0, one, one, one, None), b"logits")
    refused(lib.qw_moe_route_scored_backward(one, None, one, None, 4, 8, 2, 0, 1, 1.0, one, None), b"top_idx")
    refused(lib.qw_moe_route_scored_backward(None, one, one, None, 4, 8, 2, 0, 1, 1.0, one, None), b"scores")
    refused(lib.qw_mx_quantize(one, 7, 4, 64, 64, one, one, None), b"dtype")
    refused(lib.qw_mx_quantize(one, 0, 4, 0, 64, one, one, None), b"cols")
    refused(lib.qw_mx_quantize(one, 0, 4, 64, -1, one, one, None), b"stride")
    refused(lib.qw_mx_quantize(one, 0, 4, 64, 64, 72, one, None), b"16 bytes")
    refused(lib.qw_mx_dequantize(one, 66, 4, 64, one, 0, None), b"on 4")
    refused(lib.qw_mx_matmul(one, 1, 64, 4, None, one, 8, 64, one, None, 0, None), b"weight")
    refused(lib.qw_mx_matmul(one, 1, 64, -1, one, one, 8, 64, one, None, 0, None), b"rows")
    weights = [one] * 6
    refused(lib.qw_mx_experts(one, 1, 64, one, 2, 64, 64, -1, 0, *weights, 0, one, one, 1 << 30, None), b"rows")
    refused(lib.qw_mx_experts(one, 1, -64, one, 2, 64, 64, 4, 0, *weights, 0, one, one, 1 << 30, None), b"strides")
    refused(lib.qw_mx_experts(one, 1, 64, one, 0, 64, 64, 4, 0, *weights, 0, one, one, 1 << 30, None), b"experts")
    need = lib.qw_mx_experts_workspace_bytes(4, 2, 64, 64)
    assert lib.qw_mx_experts(one, 1, 64, one, 2, 64, 64, 4, 0, *weights, 0, one, one, need - 1,
                             None) == _lib.QW_ERR_WORKSPACE
    need = lib.qw_mx_matmul_backward_workspace_bytes(4, 8, 64, 1)
    assert lib.qw_mx_matmul_backward(one, 1, 4, one, one, 8, 64, one, one, need - 1, None) == _lib.QW_ERR_WORKSPACE
    # nothing to do is no error
    assert lib.qw_mx_quantize(None, 0, 0, 64, 64, None, None, None) == _lib.QW_OK
    assert route(None, 0, 64, 2, 0, None, 8, 1, 2, 1, 1.0, None, None, None, None) == _lib.QW_OK


@pytest.mark.parametrize("dtype,size", [(_lib.QW_F32, 4), (_lib.QW_BF16, 2)])
def test_the_gradient_of_rows_alone_takes_no_room_for_that_of_the_matrix(dtype, size):
    """The matrix as numbers, and grad_out where its width is padded; no transposed copies of rows."""
    need = _lib.load().qw_mx_matmul_backward_workspace_bytes
    matrix = 7168 * 2048 * size
    assert matrix <= need(8192, 7168, 2048, dtype) <= matrix + 1024
    assert need(8192, 7001, 2048, dtype) <= matrix + 8192 * 7040 * size + 1024


def test_oracle_rounds_to_the_nearest_value_with_ties_to_even():
    x = torch.tensor([[0.25, 0.26, 0.75, 0.74, 1.25, 1.75, 2.5, 3.5, 5.0, 5.01, 7.9, -0.25, -2.5, 4.0] + [0.0] * 18])
    want = [0, 0.5, 1, 0.5, 1, 2, 2, 4, 4, 6, 6, 0, -2, 4] + [0.0] * 18
    assert ref.on_grid(x)[0].tolist() == want
    assert ref.quantize(x)[1].tolist() == [[127, 0, 0, 0]]


def test_oracle_values_and_quantise_are_inverse():
    codes, scales = ref.stored(torch.Generator().manual_seed(3), 5, 256)
    codes[:, ::16] = 0x77  # every block reaches 6, so its scale is the stored one
    v = ref.values(codes, scales, 256)
    assert torch.equal(ref.on_grid(v), v)


@pytest.mark.parametrize("lead", [(5,), (2, 3)])
def test_a_captured_forward_is_taken_and_its_backward_refused_beside_a_graph_of_another_stream(monkeypatch, lead):
    """Through the operators, with streams, capture, device check and launches stood in for."""
    from quantaweave_amd import _hip

    now = {"stream": 1, "capturing": False}
    monkeypatch.setattr(_hip, "stream", lambda device: now["stream"])
    monkeypatch.setattr(_hip, "call_on", lambda *args: None)
    monkeypatch.setattr(_hip, "require_device", lambda t, what: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now["capturing"])
    w = ref.stored(torch.Generator().manual_seed(0), 8, 64)
    for what, op in (("mx_matmul", lambda t: qa.mx_matmul(t, *w)), ("route_experts", lambda t: qa.route_experts(t, 2)[1])):
        leaf = torch.randn(*lead, 64, requires_grad=True)
        now.update(stream=1, capturing=False)
        kept = op(leaf)  # the eager graph
        now.update(stream=7, capturing=True)
        y = op(leaf)     # a forward pass alone is no fault
        with pytest.raises(RuntimeError, match=f"{what}.*another stream"):
            torch.autograd.grad(y, leaf, torch.ones_like(y), retain_graph=True)
        now.update(capturing=False)
        assert torch.autograd.grad(y, leaf, torch.ones_like(y))[0].shape == leaf.shape  # no capture: torch's own waits do
        now.update(stream=1, capturing=True)
        y = op(leaf)
        torch.autograd.grad(y, leaf, torch.ones_like(y))  # captured on the stream the graph was made on
        del kept, y
        now.update(stream=7)
        y = op(leaf)     # the graph is gone, and its node with it
        torch.autograd.grad(y, leaf, torch.ones_like(y))


@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_tangents_are_refused(monkeypatch, requires_grad):
    """Before any launch; the device check is passed over, nothing else of the calls."""
    from torch.autograd import forward_ad

    from quantaweave_amd import _hip

    monkeypatch.setattr(_hip, "require_device", lambda t, what: None)
    x = torch.randn(4, 64, requires_grad=requires_grad)
    gen = torch.Generator().manual_seed(0)
    wide, stack, down = (ref.stored(gen, *s) for s in ((8, 64), (2, 32, 64), (2, 64, 32)))
    calls = [lambda t: qa.mx_matmul(t, *wide), lambda t: qa.route_experts(t, 2)]
    if not requires_grad:
        calls.append(lambda t: qa.mx_grouped_swiglu(t, stack, stack, down, torch.tensor([0, 1, 4]).int()))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.randn(4, 64))
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(dual)


def test_backward_under_capture_is_refused_while_a_graph_of_another_stream_lives(monkeypatch):
    """The streams and the capture are stood in for: the refusal is decided on the host, before any launch."""
    from quantaweave_amd import _hip

    now = {"stream": 1, "capturing": False}
    monkeypatch.setattr(_hip, "stream", lambda device: now["stream"])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now["capturing"])
    leaf = torch.randn(3, requires_grad=True)
    for t in (leaf, leaf * 2):
        now.update(stream=1, capturing=False)
        _hip.note_stream(t, "op")
        kept = t * 2  # the eager graph
        now.update(stream=7, capturing=True)
        with pytest.raises(RuntimeError, match="another stream"):
            _hip.note_stream(t, "op")
        now.update(stream=1)
        _hip.note_stream(t, "op")  # captured on the stream the graph was made on
        del kept
    del t
    now.update(stream=7)
    _hip.note_stream(leaf, "op")  # the graph is gone, and its node with it
