"""Tensor subclasses that no group has sharded, for the tests of the list passes."""

from __future__ import annotations

import torch


class PairTensor(torch.Tensor):
    """A value kept in two tensors of its shape; ops run on both.  ``device`` is what the wrapper claims."""

    @staticmethod
    def __new__(cls, a: torch.Tensor, b: torch.Tensor, device=None) -> "PairTensor":
        return torch.Tensor._make_wrapper_subclass(
            cls, a.shape, strides=a.stride(), dtype=a.dtype, device=a.device if device is None else device,
            requires_grad=False,
        )

    def __init__(self, a: torch.Tensor, b: torch.Tensor, device=None):
        self.a, self.b, self.claimed = a, b, device

    def __repr__(self) -> str:  # type: ignore[override]
        return f"PairTensor({self.a!r}, {self.b!r})"

    def __tensor_flatten__(self):
        return ["a", "b"], None

    @staticmethod
    def __tensor_unflatten__(inner_tensors, meta, outer_size, outer_stride):
        return PairTensor(inner_tensors["a"], inner_tensors["b"])

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        def half(x, name):
            if isinstance(x, PairTensor):
                return getattr(x, name)
            return type(x)(half(y, name) for y in x) if isinstance(x, (list, tuple)) else x

        pair = [func(*half(args, n), **{k: half(v, n) for k, v in (kwargs or {}).items()}) for n in ("a", "b")]
        claimed = next((x.claimed for x in args if isinstance(x, PairTensor)), None)
        return PairTensor(*pair, claimed) if isinstance(pair[0], torch.Tensor) else pair[0]


class OwnStorage(torch.Tensor):
    """Elements in memory of its own (``as_subclass``), next to a tensor in an attribute that ``__tensor_flatten__`` names."""

    def __tensor_flatten__(self):
        return ["extra"], None

    @property
    def extra(self) -> torch.Tensor:
        return torch.zeros(3, device=self.device)
