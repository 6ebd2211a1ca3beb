"""The C++ autograd nodes of norm, router and head loss as autograd's own rules
see them: changes in place are noticed, a freed graph is refused, a retained one
runs again, and only the gradients asked for are formed."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _norm(dev, lead=(6,)):
    from lowbit.norm import layer_norm

    ins = [torch.randn(*lead, 40, device=dev).requires_grad_(True), torch.randn(40, device=dev).requires_grad_(True),
           torch.randn(40, device=dev).requires_grad_(True)]
    return ins, lambda x, w, b: layer_norm(x, w, b)


def _route(dev, lead=(6,)):
    from lowbit.router import route_tokens

    return [torch.randn(*lead, 20, device=dev).requires_grad_(True)], lambda z: route_tokens(z, 4)[1]


def _xent(dev, lead=(6,)):
    from lowbit.loss import linear_cross_entropy

    y = torch.randint(0, 90, lead, device=dev)
    ins = [torch.randn(*lead, 40, device=dev).bfloat16().requires_grad_(True),
           torch.randn(90, 40, device=dev).bfloat16().requires_grad_(True)]
    return ins, lambda x, w: linear_cross_entropy(x, w, y, reduction="none")


ALL = pytest.mark.parametrize("make", [_norm, _route, _xent])


@ALL
@pytest.mark.parametrize("lead", [(6,), (2, 3)])
def test_a_change_in_place_is_noticed(gpu_device, make, lead):
    ins, f = make(gpu_device, lead)
    # the head's hidden rows are copied in the forward: they may change
    for i in range(1 if make is _xent else 0, 1 if make is _route else 2):
        leaves = [t.detach().clone().requires_grad_(True) for t in ins]
        moved = [t * 1 for t in leaves]
        out = f(*moved)
        with torch.no_grad():
            moved[i].mul_(2)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out.sum(), leaves)


@ALL
def test_a_graph_is_used_once_unless_kept(gpu_device, make):
    ins, f = make(gpu_device)
    up = torch.randn_like(f(*ins))
    out = f(*ins)
    first = torch.autograd.grad(out, ins, up, retain_graph=True)
    again = torch.autograd.grad(out, ins, up)
    for a, b, t in zip(first, again, ins):
        assert a.shape == t.shape and a.dtype == t.dtype and torch.equal(a, b)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(out, ins, up)


@ALL
def test_gradients_asked_for_alone(gpu_device, make):
    ins, f = make(gpu_device)
    up = torch.randn_like(f(*ins))
    every = torch.autograd.grad(f(*ins), ins, up)
    for i, t in enumerate(ins):
        (one,) = torch.autograd.grad(f(*ins), t, up)
        assert torch.equal(one, every[i])
        alone = [u if j == i else u.detach() for j, u in enumerate(ins)]
        f(*alone).backward(up)
        assert torch.equal(t.grad, every[i]) and all(u.grad is None for j, u in enumerate(ins) if j != i)
        t.grad = None


@ALL
def test_outputs_may_change_in_place_and_graphs_join(gpu_device, make):
    """the result is an ordinary part of a graph: it may be scaled in place, hooked, and used twice"""
    ins, f = make(gpu_device)
    up = torch.randn_like(f(*ins))
    every = torch.autograd.grad(f(*ins), ins, up)
    out = f(*ins)
    assert out.requires_grad and not out.is_leaf and "Backward" in out.grad_fn.name()
    seen = []
    out.register_hook(lambda g: seen.append(g.clone()))
    got = torch.autograd.grad((out * 0.5 + out * 0.5), ins, up)
    assert len(seen) == 1 and torch.allclose(seen[0], up)
    for a, b in zip(got, every):
        assert torch.allclose(a.float(), b.float(), rtol=2.0 ** -7, atol=1e-6)
    scaled = f(*ins).mul_(2.0)  # 2 is exact in every type
    for a, b in zip(torch.autograd.grad(scaled, ins, up / 2), every):
        assert torch.equal(a, b)
    with torch.no_grad():
        assert not f(*ins).requires_grad
    with torch.inference_mode():
        assert f(*ins).is_inference()
    assert not f(*[t.detach() for t in ins]).requires_grad


def test_ids_are_not_differentiable(gpu_device):
    from lowbit.router import route_tokens

    ids, w = route_tokens(torch.randn(5, 12, device=gpu_device, requires_grad=True), 3)
    assert not ids.requires_grad and w.requires_grad


def _row(dev, n, dtype=torch.float32):
    """[1, n] of strides (1, 1), as a column's transposition gives it"""
    t = torch.randn(n, 1, device=dev).to(dtype).t()
    assert t.stride() == (1, 1)
    return t


def test_one_row_of_any_pitch(gpu_device):
    """a single row has no pitch, whatever its stride says: inputs and incoming gradients"""
    from lowbit.loss import linear_cross_entropy
    from lowbit.norm import layer_norm
    from lowbit.router import route_tokens

    def same(f, *ins, up):
        got, want = [], []
        for out, plain in ((got, False), (want, True)):
            leaves = [(t.clone(memory_format=torch.contiguous_format).reshape(-1).reshape(t.shape) if plain else t)
                      .detach().requires_grad_(True) for t in ins]
            r = f(*leaves)
            u = up.reshape(-1).reshape(r.shape) if plain else up
            out += [r.detach(), *torch.autograd.grad(r, leaves, u)]
            with torch.no_grad():
                out.append(f(*leaves))
        assert all(torch.equal(a, b) for a, b in zip(got, want))

    for dtype in (torch.float32, torch.bfloat16):
        same(lambda x: layer_norm(x), _row(gpu_device, 72, dtype), up=_row(gpu_device, 72, dtype))
    same(lambda z: route_tokens(z, 4)[1], _row(gpu_device, 40), up=_row(gpu_device, 4))
    y = torch.zeros(1, dtype=torch.int64, device=gpu_device)
    w = torch.randn(90, 64, device=gpu_device).bfloat16()
    one = torch.ones(1, device=gpu_device)
    same(lambda x, w: linear_cross_entropy(x, w, y, reduction="none"), _row(gpu_device, 64, torch.bfloat16), w, up=one)
    x = torch.randn(1, 64, device=gpu_device).bfloat16()
    same(lambda x, w: linear_cross_entropy(x, w, y, reduction="none"), x, _row(gpu_device, 64, torch.bfloat16), up=one)


@ALL
def test_forward_mode_is_refused(gpu_device, make):
    """a tangent that comes with an input, or with the incoming gradient, is not dropped without a word"""
    import torch.autograd.forward_ad as fwd

    ins, f = make(gpu_device)
    up = torch.randn_like(f(*ins))
    with fwd.dual_level():
        for i in range(len(ins)):
            for leaf in (ins[i], ins[i].detach()):
                dual = [fwd.make_dual(leaf, torch.ones_like(leaf)) if j == i else t for j, t in enumerate(ins)]
                with pytest.raises(NotImplementedError, match="forward mode"):
                    f(*dual)
                with torch.no_grad(), pytest.raises(NotImplementedError, match="forward mode"):
                    f(*dual)
        out = f(*ins)
        with pytest.raises(NotImplementedError, match="forward mode"):
            torch.autograd.grad(out, ins, fwd.make_dual(up, torch.ones_like(up)))
    f(*ins).backward(up)  # and outside it they run again


@ALL
@pytest.mark.parametrize("lead", [(5, 7), (3, 4, 2)])
def test_leading_axes_in_another_order(gpu_device, make, lead):
    """rows that no view puts one behind the other (the sequence in front of the batch, as a transposition leaves it):
    gradients of the input's own shape, equal to those of its copy"""
    ins, f = make(gpu_device, lead)
    first = ins[0].detach().transpose(0, 1).contiguous().transpose(0, 1)
    assert not first.is_contiguous() and torch.equal(first, ins[0].detach())
    up = torch.randn_like(f(*ins))
    turned = up.transpose(0, 1).contiguous().transpose(0, 1)
    want = torch.autograd.grad(f(*ins), ins, up)
    leaves = [first.requires_grad_(True), *ins[1:]]
    out = f(*leaves)
    assert torch.equal(out.detach(), f(*ins).detach())
    for u in (up, turned):
        for a, b in zip(torch.autograd.grad(out, leaves, u, retain_graph=True), want):
            assert a.shape == b.shape and torch.equal(a, b)


@ALL
@pytest.mark.parametrize("which", ["host", "type", "shorter", "nothing"])
def test_other_tensors_than_those_kept_are_refused(gpu_device, make, which):
    """the kernels take the kept tensors by address: what saved-tensor hooks hand back is looked at first"""
    change = {"host": lambda t: t.cpu(), "type": lambda t: t.to(torch.float64), "shorter": lambda t: t[:-1],
              "nothing": lambda t: t.new_empty(0)}[which]
    ins, f = make(gpu_device)
    up = torch.randn_like(f(*ins))
    kinds = []

    def pack(t):
        kinds.append(t.dtype)
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        f(*ins)
    for n in range(len(kinds)):
        seen = []

        def nth(t):
            seen.append(t)
            return len(seen) - 1

        with torch.autograd.graph.saved_tensors_hooks(nth, lambda i: change(seen[i]) if i == n else seen[i]):
            out = f(*ins)
        with pytest.raises(RuntimeError, match="kept for the backward"):
            torch.autograd.grad(out, ins, up)


@ALL
def test_kept_tensors_may_come_back_in_another_layout(gpu_device, make):
    ins, f = make(gpu_device)
    up = torch.randn_like(f(*ins))
    want = torch.autograd.grad(f(*ins), ins, up)

    def spread(t):  # every element behind an unused one
        wide = torch.full((*t.shape, 2), 7, dtype=t.dtype, device=t.device)
        wide[..., 1] = t
        return wide[..., 1]

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, spread):
        out = f(*ins)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, ins, up), want))


@ALL
def test_what_the_backward_reads_passes_the_hooks(gpu_device, make):
    """saved-tensor hooks see all that a node keeps, and it may have been elsewhere in between"""
    ins, f = make(gpu_device, (700,))
    up = torch.randn_like(f(*ins))
    want = torch.autograd.grad(f(*ins), ins, up)
    kept = []

    def pack(t):
        kept.append(t.numel() * t.element_size())
        return t.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.to(gpu_device)):
        out = f(*ins)
    got = torch.autograd.grad(out, ins, up)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # norm: x, weight, bias and two numbers a row; routing: logits and ids; head: weight and the live rows with their numbers
    least = {_norm: 700 * 40 * 4 + 2 * 40 * 4 + 700 * 8, _route: 700 * 20 * 4 + 700 * 4 * 4, _xent: 90 * 40 * 2 + 700 * 64 * 2}
    assert sum(kept) >= least[make]


def test_a_checkpoint_keeps_no_hidden_rows(gpu_device):
    """recomputed in the backward, the head loss holds nothing of the rows' size until then"""
    from torch.utils.checkpoint import checkpoint

    from lowbit.loss import linear_cross_entropy

    x = torch.randn(4096, 1024, device=gpu_device).bfloat16().requires_grad_(True)
    w = torch.randn(64, 1024, device=gpu_device).bfloat16().requires_grad_(True)
    y = torch.randint(0, 64, (4096,), device=gpu_device)
    want = torch.autograd.grad(linear_cross_entropy(x, w, y), (x, w))
    before = torch.cuda.memory_allocated()
    loss = checkpoint(linear_cross_entropy, x, w, y, use_reentrant=False)
    assert torch.cuda.memory_allocated() - before < 1 << 20
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, (x, w)), want))
