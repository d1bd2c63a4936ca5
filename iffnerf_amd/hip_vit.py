"""The image backbone on the matrix cores: DINOv2 ViT-S/14 ``forward_features`` through ``iff_vit_forward``.

``ViTHandle`` owns the weight slab of one network; ``serve_natively`` installs the native ``forward_features`` ON a backbone module
(DINOv2's ``dinov2_vits14`` from ``torch.hub`` -- reference pose_estimation/backbone.py:12-14 -- or the seeded stand-in of this
package's backbone.py) so that ``forward_features(x)["x_norm_patchtokens"]`` (what pose_estimation/identification_module.py:141
reads) runs in libiffnerf_hip under ``torch.no_grad`` while the module -- class, parameters, ``state_dict`` keys -- stays what the
reference's ``create_backbone`` returns; with autograd enabled on a trainable backbone the module's own torch forward runs.
State-dict keys of both sources are understood (``blocks.i.attn.qkv.*``, ``blocks.i.ls1.gamma``, ``blocks.i.mlp.fc1.*`` for
DINOv2; ``blocks.i.qkv.*``, ``blocks.i.ls1``, ``blocks.i.fc1.*`` for the stand-in).

``train_natively`` is the counterpart for that torch forward: the layer norms, gated feed-forwards and dropouts inside a backbone run their
forward AND backward passes on ``hip_block``'s operators.
"""
from __future__ import annotations

import ctypes as C
import math
import operator
from typing import Dict, Optional

import torch
import torch.fx
import torch.nn.functional as F

from . import _lib, hip_block
from ._lib import check, dptr, stream_ptr


def interpolate_pos_embed(pos: torch.Tensor, gh: int, gw: int, patch: int = 14, differentiable: bool = False) -> torch.Tensor:
    """DINOv2's ``interpolate_pos_encoding`` for an input of gh x gw patches: ``pos`` [1, 1 + n, D] -> [1 + gh*gw, D].  The class
    position is kept; the patch grid is resized bicubically with the +0.1 scale-factor offset of the original implementation."""
    pos = pos.float() if differentiable else pos.detach().float()
    n = pos.shape[1] - 1
    if n == gh * gw:
        return pos[0].contiguous()
    side = int(round(math.sqrt(n)))
    if side * side != n:
        raise RuntimeError(f"position embedding has {n} patch positions: not a square grid")
    grid = pos[0, 1:].reshape(1, side, side, -1).permute(0, 3, 1, 2)
    grid = F.interpolate(grid, scale_factor=((gh + 0.1) / side, (gw + 0.1) / side), mode="bicubic")
    if grid.shape[-2:] != (gh, gw):
        raise RuntimeError("interpolated position grid has the wrong size")
    return torch.cat((pos[0, :1], grid.permute(0, 2, 3, 1).reshape(gh * gw, -1)), dim=0).contiguous()


PRECISIONS = {"fp32": _lib.VIT_FP32, "bf16": _lib.VIT_BF16}


def _pick(sd: Dict[str, torch.Tensor], *names):
    for n in names:
        if n in sd:
            return sd[n]
    raise RuntimeError(f"backbone state_dict has none of {names}")


DEFAULT_GEMM_FORM = 0     # iff_vit_desc.gemm_form of the handles a served backbone builds (0: the library's choice; development scripts set others for A/B runs)


class ViTHandle:
    """One ViT-S/14's weights on one GPU (``iff_vit``)."""

    def __init__(self, state_dict: Dict[str, torch.Tensor], device, grid=(16, 16), patch: int = 14, heads: int = 6, ln_eps: float = 1e-6,
                 precision: str = "fp32", gemm_form: int = 0):
        """``gemm_form`` (``iff_vit_desc.gemm_form``): 0 the library's choice of GEMM kernels; 1-4 name one (A/B runs, the bit-equality test).
        ``precision``: "fp32" (the default) -- the accuracy class of the reference's fp32 DINOv2: every matrix operand split exactly
        into two fp16 pieces, three MFMA products per block, fp32 accumulation (include/iffnerf_hip.h IFF_VIT_FP32); "bf16" -- bf16
        operands, ~2x faster, token features move by ~1e-2 relative (a throughput option)."""
        self._h = None
        if precision not in PRECISIONS:
            raise RuntimeError(f"precision must be one of {sorted(PRECISIONS)} (got {precision!r})")
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError(f"ViTHandle needs a GPU device (got {device}); libiffnerf_hip has no CPU path")
        sd = {k: v.detach() for k, v in state_dict.items()}
        depth = 1 + max(int(k.split(".")[1]) for k in sd if k.startswith("blocks."))
        dim = int(_pick(sd, "cls_token").shape[-1])
        gh, gw = int(grid[0]), int(grid[1])

        def stack(*alts):
            return torch.stack([_pick(sd, *(a.format(i=i) for a in alts)).float() for i in range(depth)])

        t = {
            "patch_w": _pick(sd, "patch_embed.proj.weight", "patch_embed.weight").float().reshape(dim, -1),
            "patch_b": _pick(sd, "patch_embed.proj.bias", "patch_embed.bias").float(),
            "cls": _pick(sd, "cls_token").float().reshape(dim),
            "pos": interpolate_pos_embed(_pick(sd, "pos_embed"), gh, gw, patch),
            "ln1_w": stack("blocks.{i}.norm1.weight"), "ln1_b": stack("blocks.{i}.norm1.bias"),
            "qkv_w": stack("blocks.{i}.attn.qkv.weight", "blocks.{i}.qkv.weight"),
            "qkv_b": stack("blocks.{i}.attn.qkv.bias", "blocks.{i}.qkv.bias"),
            "proj_w": stack("blocks.{i}.attn.proj.weight", "blocks.{i}.proj.weight"),
            "proj_b": stack("blocks.{i}.attn.proj.bias", "blocks.{i}.proj.bias"),
            "ls1": stack("blocks.{i}.ls1.gamma", "blocks.{i}.ls1"),
            "ln2_w": stack("blocks.{i}.norm2.weight"), "ln2_b": stack("blocks.{i}.norm2.bias"),
            "fc1_w": stack("blocks.{i}.mlp.fc1.weight", "blocks.{i}.fc1.weight"),
            "fc1_b": stack("blocks.{i}.mlp.fc1.bias", "blocks.{i}.fc1.bias"),
            "fc2_w": stack("blocks.{i}.mlp.fc2.weight", "blocks.{i}.fc2.weight"),
            "fc2_b": stack("blocks.{i}.mlp.fc2.bias", "blocks.{i}.fc2.bias"),
            "ls2": stack("blocks.{i}.ls2.gamma", "blocks.{i}.ls2"),
            "norm_w": _pick(sd, "norm.weight").float(), "norm_b": _pick(sd, "norm.bias").float(),
        }
        if t["patch_w"].shape[1] != 3 * patch * patch:
            raise RuntimeError(f"patch embedding has {t['patch_w'].shape[1]} inputs per patch, expected 3 x {patch} x {patch}")
        d = _lib.VitDesc()
        d.dim, d.depth, d.heads, d.mlp, d.patch, d.grid_h, d.grid_w = dim, depth, int(heads), int(t["fc1_w"].shape[1]), int(patch), gh, gw
        d.ln_eps = float(ln_eps)
        d.precision = PRECISIONS[precision]
        d.gemm_form = int(gemm_form)
        self.precision = precision
        keep = []
        for name, v in t.items():
            v = v.to(device=device, dtype=torch.float32).contiguous()
            keep.append(v)
            setattr(d, name, dptr(v, name=name))
        self.device, self.dim, self.grid, self.patch, self.depth = device, dim, (gh, gw), int(patch), depth
        out = C.c_void_p()
        with torch.cuda.device(device):
            check(_lib.lib().iff_vit_create(C.byref(d), stream_ptr(device), C.byref(out)), "iff_vit_create")
        self._h = out

    def close(self):
        if getattr(self, "_h", None):
            _lib.lib().iff_vit_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def forward(self, images: torch.Tensor, want_cls: bool = False):
        """images [Q,3,14 gh,14 gw] (resized / cropped / normalised) -> patch tokens [Q, gh*gw, dim] (+ class token [Q, dim])."""
        gh, gw = self.grid
        if images.dim() != 4 or images.shape[1] != 3 or tuple(images.shape[-2:]) != (gh * self.patch, gw * self.patch):
            raise RuntimeError(f"images must be [Q,3,{gh * self.patch},{gw * self.patch}] (got {tuple(images.shape)})")
        if not images.is_cuda:
            raise RuntimeError("images must live on the GPU; libiffnerf_hip has no CPU path")
        x = images.detach().to(torch.float32).contiguous()
        Q = x.shape[0]
        tok = x.new_empty(Q, gh * gw, self.dim)
        cls = x.new_empty(Q, self.dim) if want_cls else None
        L = _lib.lib()
        ws_bytes = int(L.iff_vit_workspace(self._h, Q))
        ws = torch.empty(max(ws_bytes, 4) // 4, dtype=torch.float32, device=x.device)
        with torch.cuda.device(self.device):
            check(L.iff_vit_forward(self._h, dptr(x), Q, dptr(tok), dptr(cls), ws.data_ptr(), ws.numel() * 4, stream_ptr(self.device)),
                  "iff_vit_forward")
        return (tok, cls) if want_cls else tok


def _drops(module: torch.nn.Module) -> bool:
    """Something in ``module`` drops values in training mode."""
    from .pose_estimation.backbone import _DropAdd
    nn = torch.nn
    kinds = (nn.Dropout, nn.Dropout1d, nn.Dropout2d, nn.Dropout3d, nn.AlphaDropout, nn.FeatureAlphaDropout, _DropAdd)
    return any(isinstance(m, kinds) and m.p > 0.0 for m in module.modules())


class _NativeForwardFeatures:
    """The callable installed as a backbone module's ``forward_features`` by ``serve_natively``.  It holds the module it serves (the
    module holds it in turn: an ordinary reference cycle) and the ``iff_vit`` handle built from the module's CURRENT parameters."""

    def __init__(self, module: torch.nn.Module, grid, patch: int, precision: str = "fp32"):
        self.module, self.grid, self.patch, self.precision = module, (int(grid[0]), int(grid[1])), int(patch), precision
        self._handles: Dict[tuple, ViTHandle] = {}        # one iff_vit per input grid (the position table is interpolated per grid)
        self._key = None

    # a handle is a device resource of THIS process: copies and pickles of the module start without one
    def __getstate__(self):
        return {"module": self.module, "grid": self.grid, "patch": self.patch, "precision": self.precision, "_handles": {}, "_key": None}

    @property
    def _handle(self) -> Optional[ViTHandle]:
        return self._handles.get(self.grid)

    def close(self):
        for h in self._handles.values():
            h.close()
        self._handles = {}

    def stock(self, x, *args, **kwargs):
        """The module's own (class-level) ``forward_features``: stock torch ops."""
        return type(self.module).forward_features(self.module, x, *args, **kwargs)

    def _vit(self, device, grid=None) -> ViTHandle:
        grid = self.grid if grid is None else (int(grid[0]), int(grid[1]))
        key = (str(device),) + tuple((p.data_ptr(), p._version) for p in self.module.parameters())
        if self._key != key:
            self.close()
            self._key = key
        if grid not in self._handles:
            self._handles[grid] = ViTHandle(self.module.state_dict(), device, grid, self.patch, precision=self.precision, gemm_form=DEFAULT_GEMM_FORM)
        return self._handles[grid]

    MAX_TOKENS = 288          # csrc/api.hip iff_vit_create: 1 + gh * gw tokens per image at most

    def __call__(self, x, masks=None, *args, **kwargs):
        if not isinstance(x, torch.Tensor) or masks is not None or args or kwargs:
            return self.stock(x, masks, *args, **kwargs)          # token masking / list inputs: DINOv2's training-side forms
        if torch.is_grad_enabled() and (x.requires_grad or any(p.requires_grad for p in self.module.parameters())):
            return self.stock(x)
        if self.module.training and _drops(self.module):
            return self.stock(x)                                  # (the kernels drop nothing)
        if x.is_cuda and x.dim() == 4:
            # any input whose sides are multiples of the patch size is served, each grid by its own handle (the hub module accepts
            # them all: it interpolates its position table, and so does ViTHandle); grids beyond the kernels' token budget run the
            # module's own forward ON THE GPU.  CPU tensors raise: libiffnerf_hip has no CPU path (tests/test_abi.py).
            gh, gw = x.shape[-2] // self.patch, x.shape[-1] // self.patch
            if (gh * self.patch, gw * self.patch) != tuple(x.shape[-2:]) or 1 + gh * gw > self.MAX_TOKENS:
                return self.stock(x)
            tok, cls = self._vit(x.device, (gh, gw)).forward(x, want_cls=True)
            return {"x_norm_clstoken": cls, "x_norm_patchtokens": tok}
        tok, cls = self._vit(x.device).forward(x, want_cls=True)
        return {"x_norm_clstoken": cls, "x_norm_patchtokens": tok}


def serve_natively(module: torch.nn.Module, grid=(16, 16), patch: int = 14, precision: str = "fp32") -> torch.nn.Module:
    """Serve ``module.forward_features`` (what pose_estimation/identification_module.py:141 calls) from ``iff_vit_forward`` and
    return THE SAME module.  Nothing is wrapped: the module keeps its class, its parameters and its ``state_dict`` keys, so an
    ``IdentificationModule`` built on it saves and strict-loads ``image_preprocessing_net.<backbone key>`` exactly as the reference
    does (train_eval_pose_est.py:59-66, pose_estimation/train.py:226).  Only the instance attribute ``forward_features`` is
    installed: no-grad inference on a GPU tensor goes through the HIP kernels (the handle is rebuilt when a parameter moves or
    changes in place); with autograd enabled on a trainable backbone, with a dropout at work (training mode), with token masks or list
    inputs the module's own torch forward runs.  ``precision``: see ``ViTHandle`` ("fp32": the reference's accuracy class, the default;
    "bf16": throughput).  ``restore_stock(module)`` removes it."""
    if precision not in PRECISIONS:
        raise RuntimeError(f"precision must be one of {sorted(PRECISIONS)} (got {precision!r})")
    if not hasattr(type(module), "forward_features"):
        raise RuntimeError(f"{type(module).__name__} has no forward_features: not a DINOv2-style backbone")
    restore_stock(module)
    object.__setattr__(module, "forward_features", _NativeForwardFeatures(module, grid, patch, precision))
    return module


def restore_stock(module: torch.nn.Module) -> torch.nn.Module:
    """Undo ``serve_natively``: ``forward_features`` is the class's method again."""
    cur = module.__dict__.get("forward_features")
    if isinstance(cur, _NativeForwardFeatures):
        cur.close()
        object.__delattr__(module, "forward_features")
    return module


def is_served_natively(module: torch.nn.Module) -> bool:
    return isinstance(module.__dict__.get("forward_features"), _NativeForwardFeatures)


# ---------------------------------------------------------------------------------------------------- training
def _autocast(*tensors):
    """What an autocast region casts the operands of a matrix product to; outside one, the tensors as they are."""
    if not torch.is_autocast_enabled("cuda"):
        return tensors
    dt = torch.get_autocast_dtype("cuda")
    return tuple(t if t is None or not t.is_floating_point() else t.to(dt) for t in tensors)


def _in_fp32(*tensors):
    """What an autocast region runs in fp32 gets 16-bit tensors as fp32 there (and answers in fp32); outside one, the tensors as they are."""
    if not torch.is_autocast_enabled("cuda"):
        return tensors
    return tuple(t.float() if t is not None and t.dtype in (torch.float16, torch.bfloat16) else t for t in tensors)


class _NativeForward:
    """The callable installed as a sub-module's ``forward`` by ``train_natively``.  It reads the module's own parameters at every call:
    optimizer steps, ``.to(...)`` and ``load_state_dict`` need nothing else."""

    def __init__(self, module: torch.nn.Module):
        self.module = module


class _NativeLayerNorm(_NativeForward):
    def __call__(self, x):
        m = self.module
        if x.shape[-1:] != m.normalized_shape:
            raise RuntimeError(f"expected an input whose last axis is {m.normalized_shape[0]} wide (normalized_shape), got shape {tuple(x.shape)}")
        return hip_block.layer_norm(*_in_fp32(x, m.weight, m.bias), m.eps)


def _same(a, b) -> bool:
    return a is b or (type(a) is type(b) and isinstance(a, (int, float, str)) and a == b)      # (after pickling a number is another object)


class _NativeGatedMlp(_NativeForward):
    count = -1                                                    # (pickled before a forward was looked at: the module's own runs)

    def __init__(self, module):
        super().__init__(module)
        d = module.__dict__
        self.children = tuple(module._modules.values())
        self.others = tuple(c for c in self.children if c is not module.w12 and c is not module.w3)
        self.attributes = tuple((k, v) for k, v in d.items() if k not in ("training", "forward") and not k.startswith("_"))
        self.count = len(d) - ("forward" in d)

    def __call__(self, x):
        m = self.module
        # what the module's forward was shown to compute holds for what it could go by then: hooks, children or attributes that came or
        # changed since are the module's own forward's to deal with
        if not (len(m.__dict__) == self.count + 1 and tuple(m._modules.values()) == self.children and _just_linear(m.w12) and _just_linear(m.w3)
                and all(_same(m.__dict__.get(k), v) for k, v in self.attributes) and all(c is None or _passes(c) for c in self.others)):
            return type(m).forward(m, x)
        return hip_block.gated_mlp(*_autocast(x, m.w12.weight, m.w12.bias, m.w3.weight, m.w3.bias))


def _fresh_seed(x: torch.Tensor) -> torch.Tensor:
    # one value of torch's own generator on the device: follows torch.manual_seed, is replayed by activation checkpointing, and a
    # captured step draws another one at every replay
    return torch.empty(1, dtype=torch.int64, device=x.device).random_()


class _NativeDropout(_NativeForward):
    def __call__(self, x):
        m = self.module
        return hip_block.dropout(x, m.p, _fresh_seed(x)) if m.training and m.p > 0.0 else x


class _NativeDropAdd(_NativeForward):
    def __call__(self, residual, branch):
        m = self.module
        if not (m.training and m.p > 0.0):
            return residual + branch
        if residual.shape != branch.shape:                        # (a sum that broadcasts)
            return residual + hip_block.dropout(branch, m.p, _fresh_seed(branch))
        dt = torch.promote_types(residual.dtype, branch.dtype)
        return hip_block.dropout(branch.to(dt), m.p, _fresh_seed(branch), residual=residual.to(dt))


def _runs(m, cls) -> bool:
    """m computes what ``cls`` computes: that class or a subclass without a forward of its own, and none installed on the instance."""
    return isinstance(m, cls) and type(m).forward is cls.forward and isinstance(m.__dict__.get("forward"), (type(None), _NativeForward))


def _unwatched(m) -> bool:
    return not (m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks)


def _just_linear(m) -> bool:
    """m is its weight and bias and nothing else: no hook would see, or change (weight norm), what a call that skips it computes."""
    return _runs(m, torch.nn.Linear) and _unwatched(m)


def _passes(c) -> bool:
    """A child beside ``w12`` and ``w3`` that a call may skip: SiLU, or the identity."""
    return _unwatched(c) and ((_runs(c, torch.nn.SiLU) and not c.inplace) or _runs(c, torch.nn.Identity) or (_runs(c, torch.nn.Dropout) and c.p == 0.0))


class _Watch(torch.fx.Tracer):
    """Every child is a leaf; no operation is recorded outside the modes the trace began in (a ``no_grad`` or ``autocast`` inside the
    forward is no operation itself)."""

    def __init__(self):
        super().__init__()
        self.modes = self._modes()

    @staticmethod
    def _modes():
        return (torch.is_grad_enabled(), torch.is_inference_mode_enabled(), torch.is_autocast_enabled("cuda"), torch.get_autocast_dtype("cuda"))

    def is_leaf_module(self, m, name):
        return True

    def create_node(self, *args, **kwargs):
        if self._modes() != self.modes:
            raise RuntimeError("an operation under modes of its own")
        return super().create_node(*args, **kwargs)


def _is_gated_silu_graph(m: torch.nn.Module, graph) -> bool:
    """The traced operations are ``w3(silu(gate) * up)`` of ``[gate | up] = w12(x)``: each value is what it must be, and used once."""
    half, value = m.w3.in_features, {}

    def bound(node, *names):
        return {**dict(zip(names, node.args)), **node.kwargs}

    for n in graph.nodes:
        users = 1
        if n.op == "placeholder":
            new = "x" if not value and not str(n.target).startswith("*") and not n.args else None
        elif n.op == "call_module":
            child, a = m.get_submodule(n.target), bound(n, "input")
            of = value.get(a.pop("input", a.pop("x", None))) if len(a) == 1 else None
            if child is m.w12:
                new = "both" if of == "x" else None
                users = 2 if len(n.users) == 2 else 1                  # (two slices, or one chunk)
            elif child is m.w3:
                new = "y" if of == "hidden" else None
            elif _runs(child, torch.nn.SiLU):
                new = "act" if of == "gate" else None
            else:
                new = of if _passes(child) else None
        elif (n.op, n.target) in (("call_method", "chunk"), ("call_function", torch.chunk), ("call_method", "split"), ("call_function", torch.split)):
            size = "chunks" if n.target in ("chunk", torch.chunk) else "split_size"
            a = bound(n, "of", size, "dim")
            a.setdefault("of", a.pop("input", a.pop("tensor", None)))
            right = set(a) == {"of", size, "dim"} and a[size] == (2 if size == "chunks" else half) and a["dim"] == -1
            new = "halves" if right and value.get(a["of"]) == "both" else None
            users = 2
        elif (n.op, n.target) == ("call_function", operator.getitem) and len(n.args) == 2 and not n.kwargs:
            of, at = value.get(n.args[0]), n.args[1]
            new = None
            if of == "halves":
                new = {0: "gate", 1: "up"}.get(at)
            elif of == "both" and isinstance(at, tuple) and len(at) == 2 and at[0] is Ellipsis and isinstance(at[1], slice) and at[1].step is None:
                new = {(None, half): "gate", (0, half): "gate", (half, None): "up", (half, 2 * half): "up"}.get((at[1].start, at[1].stop))
        elif (n.op, n.target) == ("call_function", F.silu):
            a = bound(n, "input", "inplace")
            new = "act" if value.get(a.pop("input", None)) == "gate" and not a.pop("inplace", False) and not a else None
        elif n.op in ("call_function", "call_method") and n.target in (operator.mul, torch.mul, "mul") and len(n.args) == 2 and not n.kwargs:
            new = "hidden" if sorted(str(value.get(v)) for v in n.args if isinstance(v, torch.fx.Node)) == ["act", "up"] else None
        elif n.op == "output":
            return len(n.args) == 1 and isinstance(n.args[0], torch.fx.Node) and value.get(n.args[0]) == "y"
        else:
            new = None
        if new is None or len(n.users) != users:
            return False
        value[n] = new
    return False


def _computes_gated_silu(m: torch.nn.Module) -> bool:
    """What m's own forward does, by tracing it in training and evaluation, with and without gradients and autocast; a forward that cannot be
    traced, takes more than its input, goes by the input's shape or values, or leaves something behind in the module does not count."""
    before, training = dict(m.__dict__), m.training
    cast, dtype = torch.is_autocast_enabled("cuda"), torch.get_autocast_dtype("cuda")
    try:
        torch.set_autocast_dtype("cuda", torch.bfloat16)
        for mode in range(8):
            m.training = bool(mode & 1)
            torch.set_autocast_enabled("cuda", bool(mode & 2))
            with torch.set_grad_enabled(bool(mode & 4)):
                if not _is_gated_silu_graph(m, _Watch().trace(m)):
                    return False
        m.training = training
        return list(m.__dict__) == list(before) and all(v is before[k] for k, v in m.__dict__.items())
    except Exception:                            # (whatever a forward raises on a tensor that is none)
        return False
    finally:
        torch.set_autocast_enabled("cuda", cast)
        torch.set_autocast_dtype("cuda", dtype)
        m.__dict__.clear()
        m.__dict__.update(before)


def _is_gated_silu(m: torch.nn.Module) -> bool:
    """``w12`` and ``w3`` of matching widths, nothing else that learns or keeps state, and a forward that is the gated SiLU block."""
    w12, w3 = getattr(m, "w12", None), getattr(m, "w3", None)
    if not (_just_linear(w12) and _just_linear(w3) and w12.out_features == 2 * w3.in_features):
        return False
    if not isinstance(m.__dict__.get("forward"), (type(None), _NativeForward)) or m._parameters or m._buffers:
        return False
    if not all(c is None or c is w12 or c is w3 or _passes(c) for c in m.children()):
        return False
    return _computes_gated_silu(m)


def _native_forward(m: torch.nn.Module):
    from .pose_estimation.backbone import _DropAdd
    if _runs(m, torch.nn.LayerNorm) and len(m.normalized_shape) == 1:
        return _NativeLayerNorm(m)
    if _runs(m, torch.nn.Dropout) and not m.inplace:
        return _NativeDropout(m)
    if _runs(m, _DropAdd):
        return _NativeDropAdd(m)
    if _is_gated_silu(m):
        return _NativeGatedMlp(m)
    return None


def train_natively(module: torch.nn.Module) -> torch.nn.Module:
    """Run the layer norms, gated feed-forwards (``w12`` / ``w3`` as in DINOv2, SiLU) and dropouts inside ``module`` -- a backbone that
    pose_estimation/train.py:97-119 back-propagates through -- on ``hip_block``'s operators, forward and backward, and return THE SAME
    module.  As with ``serve_natively`` nothing is wrapped: classes, parameters and ``state_dict`` keys stay, one instance attribute
    ``forward`` per sub-module is installed.  The module then needs GPU tensors; values differ from stock torch by rounding, and a dropout's
    mask comes from another generator (seeded by torch's).  A norm or dropout with a forward of its own is left as it is, and so is every
    feed-forward whose forward a symbolic trace does not show to be ``w3(silu(gate) * up)`` of ``[gate | up] = w12(x)``.
    ``train_stock(module)`` removes it; without this call nothing changes."""
    for m in module.modules():
        f = _native_forward(m)
        if f is not None:
            object.__setattr__(m, "forward", f)
    return module


def train_stock(module: torch.nn.Module) -> torch.nn.Module:
    """Undo ``train_natively``: every sub-module's ``forward`` is its class's method again."""
    for m in module.modules():
        if isinstance(m.__dict__.get("forward"), _NativeForward):
            object.__delattr__(m, "forward")
    return module
