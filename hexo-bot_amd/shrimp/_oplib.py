"""Registration of differentiable ``shrimp::`` operators with little between the
call and the launch.

``torch.library.custom_op`` costs a small call a third of its time, and its
generated autograd some 60 us per forward and backward; an operator defined here
has one Python kernel, and at the autograd key one ``torch.autograd.Function``,
applied only when a gradient is wanted. The public functions go past the
dispatcher where nothing listens there (``direct``), and a Function's backward
starts from its forward's argument struct: it runs on autograd's own thread,
where every line of Python costs three times as much.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

_LIB = torch.library.Library("shrimp", "FRAGMENT")


def define(schema: str, kernel, fake, function=None):
    """Defines ``shrimp::<schema>``, returns its overload. ``kernel`` runs it (for every
    device: it refuses what is not on a ROCm one), ``fake`` gives the shapes; ``function``
    is a torch.autograd.Function class whose apply takes the operator's arguments, all of
    them, and whose forward calls the overload below autograd (``below``)."""

    name = schema[: schema.index("(")]
    _LIB.define(schema)
    _LIB.impl(name, kernel, "CompositeExplicitAutograd")
    torch.library.register_fake(f"shrimp::{name}")(fake)
    op = getattr(torch.ops.shrimp, name).default
    if function is not None:

        def autograd(*args):
            if forward_ad._current_level >= 0 and any(
                isinstance(a, torch.Tensor) and forward_ad.unpack_dual(a).tangent is not None for a in args
            ):
                raise RuntimeError(f"shrimp::{name} has no forward-mode derivative")
            if torch.is_grad_enabled() and any(
                isinstance(a, torch.Tensor) and a.requires_grad for a in args
            ):
                return function.apply(*args)
            with torch._C._AutoDispatchBelowAutograd():
                return op(*args)

        _LIB.impl(name, autograd, "Autograd")
    return op


def direct(*tensors) -> bool:
    """Plain tensors, no tracing, dispatch mode or forward-mode level: a kernel may be called
    as it is."""

    if (torch.compiler.is_compiling() or torch._C._len_torch_dispatch_stack()
            or forward_ad._current_level >= 0 or torch._C._is_tracing()):
        return False
    for t in tensors:
        if type(t) is not torch.Tensor and type(t) is not torch.nn.Parameter:
            return False
    return True


def wants_grad(*tensors) -> bool:
    if not torch.is_grad_enabled():
        return False
    for t in tensors:
        if t.requires_grad:
            return True
    return False


def below(op, *args):
    """op(*args) without its autograd kernel."""

    with torch._C._AutoDispatchBelowAutograd():
        return op(*args)


def hooked() -> bool:
    """Saved tensors go through a hook (checkpointing, offloading): a backward gets others
    than its forward had, and the forward's may be gone, so it starts anew from them."""

    return torch._C._autograd._top_saved_tensors_default_hooks(True) is not None


def places(tensors):
    """Where tensors lie. A backward starts from its forward's argument struct only if all
    that it saved lies where it did (a hook may also have been put on the node itself)."""

    return [t.data_ptr() for t in tensors]


def copies(laid, given):
    """The tensors laid out anew for a launch: a backward holds these beside what it saved."""

    return tuple(a for a, b in zip(laid, given) if a is not b)


def check_sizes(what: str, name: str, t: torch.Tensor) -> None:
    if max(t.shape) >= 2**31:
        raise ValueError(f"{what}: {name} {tuple(t.shape)}, sizes below 2^31 expected")
