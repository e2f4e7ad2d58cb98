"""What the torch entry points of the grouped products and of the orthogonalised update do beside autograd: they record nothing, so
operands that require a gradient are refused while it records, and what they overwrite counts as changed."""
import pytest

torch = pytest.importorskip("torch")


def _lib():
    from gp_amd import lib
    return lib


def calls(device, wants):
    """The three entry points on small tensors; `wants`: which of their operands requires a gradient."""
    lib = _lib()
    z = lambda name, *s: torch.zeros(*s, device=device, requires_grad=name == wants)  # noqa: E731
    off = torch.tensor([0, 2, 4], device=device)
    return [lambda: lib.grouped_gemm(z("a", 4, 8), z("b", 2, 6, 8), off, z("out", 4, 6)),
            lambda: lib.grouped_gemm_dw(z("a", 4, 8), z("b", 4, 6), off, z("out", 2, 6, 8)),
            lambda: lib.orthogonalize(z("a", 4, 8), z("out", 4, 8))]


@pytest.mark.parametrize("wants", ["a", "b", "out"])
def test_operands_that_require_a_gradient_are_refused(wants):
    for call in calls("cpu", wants)[:2 if wants == "b" else 3]:
        with pytest.raises(ValueError, match="autograd"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="on the GPU"):   # the next thing that is wrong with them
            call()


@pytest.mark.gpu
def test_they_are_taken_without_recording():
    for wants in ("a", "b", "out"):
        for call in calls("cuda", wants):
            with torch.no_grad():
                assert call().grad_fn is None
            with torch.inference_mode():
                call()


@pytest.mark.gpu
def test_a_backward_pass_that_saved_what_is_overwritten_raises():
    lib = _lib()
    off = torch.tensor([0, 2, 4], device="cuda")
    r = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    for shape, write in (((4, 6), lambda out: lib.grouped_gemm(r(4, 8), r(2, 6, 8), off, out)),
                         ((2, 6, 8), lambda out: lib.grouped_gemm_dw(r(4, 8), r(4, 6), off, out)),
                         ((4, 8), lambda out: lib.orthogonalize(r(4, 8), out))):
        out, p = torch.ones(shape, device="cuda"), torch.ones(shape, device="cuda", requires_grad=True)
        loss = (out * p).sum()   # saves out
        write(out)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
