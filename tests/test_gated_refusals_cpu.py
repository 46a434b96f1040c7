"""Calls of the gated recurrence and of dropout that are refused on the host, before any
CUDA call, because their answer would be wrong."""

import pytest

torch = pytest.importorskip("torch")

import torch.autograd.forward_ad as fw  # noqa: E402

from yufmusicgen_b200.dropout import dropout  # noqa: E402
from yufmusicgen_b200.gated_scan import gated_scan, gated_scan_step  # noqa: E402


@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_tangents_are_refused(requires_grad):
    """A tangent that no derivative carries on would be lost without a word."""
    plain = {"x": torch.ones(1, 3, 4), "forget": torch.ones(1, 3, 4), "gate": torch.ones(1, 3, 4),
             "lower": torch.zeros(4), "state": torch.zeros(1, 4)}
    token = {k: t[:, 0] if t.dim() == 3 else t for k, t in plain.items()}
    with fw.dual_level():
        for call, args in ((gated_scan, plain), (gated_scan_step, token),
                           (lambda x, residual: dropout(x, 0.5, 1, residual=residual),
                            {"x": torch.ones(3), "residual": torch.ones(3)})):
            for k, t in args.items():
                dual = fw.make_dual(t.clone().requires_grad_(requires_grad), torch.ones_like(t))
                with pytest.raises(NotImplementedError, match="tangent"):
                    call(**{**args, k: dual})
                with torch.no_grad(), pytest.raises(NotImplementedError, match="tangent"):
                    call(**{**args, k: dual})


def test_sizes_beyond_the_limits_are_value_errors():
    """Refused before an output is allocated (the tensors here are one element, shared)."""
    one = torch.zeros(1, 1, 1)
    for shape in ((1, 2**30 + 1, 1), (2**26 + 1, 1, 1), (1, 1, 2**31), (2**20, 1, 32 * 64 + 1)):
        with pytest.raises(ValueError, match="too large"):
            gated_scan(one.expand(shape), one.expand(shape))
    big = one[0].expand(2**20, 2**18 + 1)
    with pytest.raises(ValueError, match="too large"):
        gated_scan_step(big, big, big)
    with pytest.raises(ValueError, match="too large"):
        dropout(one.expand(2**20, 2**10, 2**10 + 1), 0.5, 1)
    for shape in ((1, 2**30, 1), (2**26, 1, 1), (2**20, 1, 32 * 64)):  # at the limits
        with pytest.raises(ValueError, match="CUDA"):
            gated_scan(one.expand(shape), one.expand(shape))


def test_a_state_that_overlaps_an_input_is_refused():
    """The step reads its inputs while it writes the state: shared memory is allowed only
    element by element, and not with the gate."""
    B, D = 4, 6
    pool, other = torch.zeros(B + 3, D), torch.zeros(B, D)
    wide = torch.zeros(B + 2, 3 * D + 1)

    def refused(word, x, f, state, gate=None, lower=None):
        with pytest.raises(ValueError, match=word):
            gated_scan_step(x, f, state, gate, lower)

    state = pool[1:B + 1]
    for bad in (pool[:B], pool[2:B + 2], pool[3:B + 3], pool[2:3].expand(B, D), pool.view(-1)[D + 1:].as_strided((B, D), (D, 1)),
                pool.view(-1).as_strided((B, D), (D - 1, 1))):
        refused("share memory", bad, other, state)
        refused("share memory", other, bad, state)
        refused("share memory", other, other, state, bad)
    refused("share memory", other, other, state, None, pool[2])
    refused("share memory", wide[:B, :D], other, wide[1:B + 1, :D])
    refused("share memory", wide[:B, 1:D + 1], other, wide[:B, :D])
    refused("share memory", other[:1], other[:1], pool[:1], None, pool.view(-1)[1:D + 1])
    refused("share memory", wide.view(-1).as_strided((3, 2), (7, 1), 4), torch.zeros(3, 2), wide.view(-1).as_strided((3, 2), (14, 1), 10))
    half = torch.zeros(B, D, dtype=torch.bfloat16)
    refused("share memory", other.view(torch.bfloat16)[:, :D], half, other)
    # the gate may be read after the state has been written
    refused("share memory", other, other, state, state)
    refused("share memory", other, other, wide[:B, :D], wide[:B, :D])
    # nothing shared, or each element with itself: the next check answers
    for x, f, st, lower in ((state, other, state, None), (pool[:1], other[:1], pool[1:2], pool[2]), (state, state, state, pool[0]),
                            (wide[:B, :D], wide[:B, D:2 * D], wide[:B, 2 * D:3 * D], wide[B, :D]),
                            (pool[5:6].expand(2, D), other[:2], pool[3:5], pool[2]), (pool[:2], other[:2], pool[2:4], pool[4]),
                            (wide.view(-1).as_strided((3, 2), (7, 1), 4), torch.zeros(3, 2), wide.view(-1).as_strided((3, 2), (14, 1), 9), None),
                            (pool[2:3], other[:1], pool[2:3], pool[2]), (pool[:0], other[:0], pool[:0], None)):
        refused("CUDA", x, f, st, None, lower)


class Wrapper(torch.Tensor):
    """A tensor that says it lies on a GPU and has no memory, at an offset."""

    @staticmethod
    def __new__(cls, *shape, dtype=torch.float32):
        strides = torch.empty(shape, device="meta").stride()
        return torch.Tensor._make_wrapper_subclass(cls, shape, strides=strides, dtype=dtype, device="cuda", storage_offset=64)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError(f"{func} was called")


def test_tensors_without_memory_are_refused():
    """Their data pointers are null or a small offset: no kernel may get one."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        fake = torch.empty(2, 3, 4, device="cuda")[1:]
        low, step = torch.empty(8, device="cuda")[4:], torch.empty(2, dtype=torch.int64, device="cuda")[1:]
        cu = torch.empty(4, dtype=torch.int32, device="cuda")[1:]
    kinds = [(fake, low, cu, step), (Wrapper(1, 3, 4), Wrapper(4), Wrapper(3, dtype=torch.int32), Wrapper(1, dtype=torch.int64))]
    real = torch.zeros(1, 3, 4)
    for x, low, cu, step in kinds:
        for args in ((x, x), (real, x), (real, real, x), (real, real, None, low), (real, real, None, None, low[None] if x is fake else Wrapper(1, 4)),
                     (real, real, None, None, None, cu)):
            with pytest.raises(TypeError, match="memory"):
                gated_scan(*args)
        for args in ((x, 0.5, 1), (real, 0.5, 1, 0, x), (real, 0.5, 1, step)):
            with pytest.raises(TypeError, match="memory"):
                dropout(*args)
    x2 = Wrapper(3, 4)
    for args in ((x2, x2, x2), (real[0], real[0], x2), (real[0], real[0], real[0].clone(), x2)):
        with pytest.raises(TypeError, match="memory"):
            gated_scan_step(*args)
    with pytest.raises(TypeError, match="memory"):
        torch.vmap(lambda t: gated_scan(t, t)[0])(real[None])
    with pytest.raises(TypeError, match="memory"):
        gated_scan(real.to_sparse(), real)
    zeros = torch._efficientzerotensor((3, 4))
    with pytest.raises(ValueError, match="zeros"):
        gated_scan_step(real[0], real[0], zeros)


def test_tangents_do_not_matter_where_forward_mode_is_off():
    x = torch.ones(1, 3, 4)
    with fw.dual_level():
        dual = fw.make_dual(x, x)
        with fw._set_fwd_grad_enabled(False):
            for call in (lambda: gated_scan(dual, x), lambda: gated_scan_step(dual[0], x[0], x[0].clone()),
                         lambda: dropout(dual, 0.5, 1)):
                with pytest.raises(ValueError, match="CUDA"):  # the next refusal, on a host without a GPU
                    call()
