"""Calls of the trainable block operators that go through more of torch than the operator: hooks on saved tensors, forward-mode tangents,
autocast, modules of all kinds under ``train_natively``."""
import pytest
import torch

from iffnerf_amd import hip_block
from tests.test_hip_block import IDS, TYPES, check_norm, make_mlp, mlp_reference, norm_reference, normal, philox_bits, within

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def copied():
    """Saved tensors come back as dense copies, the way an offload or a compression hands them back."""
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t)


def turned():
    """... or with their axes the other way round in memory."""
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.permute(*reversed(range(t.dim()))).contiguous().permute(*reversed(range(t.dim()))))


# ------------------------------------------------------------------------------------------------------------ hooks on saved tensors
@pytest.mark.parametrize("hook", [copied, turned])
def test_the_norms_backward_describes_the_tensor_it_is_handed(hook, monkeypatch):
    """Without a GPU: the rows that the backward entry is told to read are the saved rows, inside the tensor (as_strided checks its bounds)."""
    x = torch.arange(3 * 5 * 4, dtype=torch.float32).view(3, 5, 4)[:, 1:].requires_grad_(True)
    seen = []

    def record(name, t, *args):
        if name == "iff_layer_norm_backward":
            n0, n1, s0, s1, D = args[2:7]
            assert args[0] == t.data_ptr()
            seen.append(t.as_strided((n0, n1, D), (s0, s1, 1)).reshape(3, 4, 4).clone())

    monkeypatch.setattr(hip_block, "_run", record)
    w = torch.ones(4, requires_grad=True)
    with hook():
        y = hip_block._LayerNorm.apply(x, w, None, 1e-6)
    torch.autograd.grad(y, (x, w), torch.ones_like(y))
    assert len(seen) == 1 and torch.equal(seen[0], x.detach())


@pytest.mark.parametrize("change", [lambda t: t.half(), lambda t: t[None]], ids=["type", "shape"])
def test_what_comes_back_as_something_else_is_refused(change, monkeypatch):
    """Without a GPU: a hook that hands back another type or shape ends in an error, not in a launch."""
    ran = []
    monkeypatch.setattr(hip_block, "_run", lambda name, *a: ran.append(name))
    x, w12, w3 = (torch.zeros(s, requires_grad=True) for s in ((3, 4), (12, 4), (5, 6)))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
        calls = [hip_block._LayerNorm.apply(x, torch.ones(4), None, 1e-6), hip_block._GatedMlp.apply(x, w12, None, w3, None, 0),
                 hip_block._Dropout.apply(x, None, 100, 0, torch.zeros(1, dtype=torch.int64), 0)]
    del ran[:]
    for y in calls:
        with pytest.raises(RuntimeError, match="came back as"):
            torch.autograd.grad(y, (x,), torch.ones_like(y))
    assert not ran


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_gradients_under_hooks_on_saved_tensors(dev, dtype):
    """save_on_cpu, copies and turned copies.  Norm over strided rows: the bounds of the plain call against 64 bits (a copy is aligned where
    the view was not, so the backward pass may take another form and add in another order).  Feed-forward and dropout: the same bits."""
    base = normal((3, 11, 48), 10, dtype)
    w, b = normal((40,), 8, dtype, 0.2, 1.0), normal((40,), 9, dtype)
    x, w12, b12, w3, b3, dy = make_mlp(20, 48, 80, 40, dtype, True, seed=50)
    few, fdy = x[:3], dy[:3]
    mlp = [t.requires_grad_(True) for t in (w12, b12, w3, b3)]
    seed = torch.tensor([7], device=dev)

    def more():
        out = []
        for inp, g in ((x, dy), (few, fdy)):
            i = inp.detach().requires_grad_(True)
            y = hip_block.gated_mlp(i, *mlp)
            out += [y, *torch.autograd.grad(y, (i, *mlp), g)]
        d = x.detach().requires_grad_(True)
        y = hip_block.dropout(d, 0.3, seed)
        return (*out, y, *torch.autograd.grad(y, (d,), torch.ones_like(y)))

    views = [base[:, 1:, :40], base[:, :, 8:], base[:, ::2, 3:43], base[:, :, :40].transpose(0, 1), base[1, :, :40], base[:1, :, :40].expand(4, 11, 40)]
    want = more()
    for hook in (torch.autograd.graph.save_on_cpu, copied, turned):
        for v in views:
            with hook():
                check_norm(v, w, b, 1e-6, normal(tuple(v.shape), 11, dtype))
        with hook():
            assert all(torch.equal(p, q) for p, q in zip(more(), want))


@gpu
def test_what_comes_back_on_another_device_is_refused(dev):
    x, w12, _, w3, _, _ = make_mlp(4, 8, 8, 8, torch.float32, False)
    x.requires_grad_(True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.cpu()):
        calls = [hip_block.layer_norm(x), hip_block.gated_mlp(x, w12, None, w3, None), hip_block.dropout(x, 0.5, torch.tensor([1], device=dev))]
    for y in calls:
        with pytest.raises(RuntimeError, match="came back as"):
            torch.autograd.grad(y, (x,), torch.ones_like(y))


# ------------------------------------------------------------------------------------------------------------ train_natively
class Ffn(torch.nn.Module):
    """w12 and w3 of matching widths; what happens between them is the subclass's."""

    def __init__(self, **more):
        super().__init__()
        self.w12, self.w3 = torch.nn.Linear(8, 12), torch.nn.Linear(6, 8)
        for name, value in more.items():
            setattr(self, name, value)


def ffn(forward, **more):
    return type("Its", (Ffn,), {"forward": forward})(**more)


def chunked(self, x):
    gate, up = self.w12(x).chunk(2, dim=-1)
    return self.w3(torch.nn.functional.silu(gate) * up)


def gelu(self, x):
    gate, up = self.w12(x).chunk(2, dim=-1)
    return self.w3(torch.nn.functional.gelu(gate) * up)


def up_first(self, x):
    up, gate = self.w12(x).chunk(2, dim=-1)
    return self.w3(torch.nn.functional.silu(gate) * up)


def scaled_and_dropped(self, x):
    gate, up = self.w12(x).chunk(2, dim=-1)
    return self.w3(torch.nn.functional.dropout(torch.nn.functional.silu(gate) * up * self.scale, 0.1, self.training))


def dropped(self, x):
    gate, up = self.w12(x).chunk(2, dim=-1)
    return self.w3(torch.nn.functional.dropout(torch.nn.functional.silu(gate) * up, self.drop, self.training))


def own_nonlinearity(self, x):
    gate, up = self.w12(x).chunk(2, dim=-1)
    return self.w3(self.nonlinearity(gate) * up)


def frozen_half(self, x):
    with torch.no_grad():
        both = self.w12(x)
    gate, up = both.chunk(2, dim=-1)
    return self.w3(torch.nn.functional.silu(gate) * up)


def in_full_precision(self, x):
    with torch.autocast("cuda", enabled=False):
        return chunked(self, x)


def training_noise(self, x):
    h = chunked(self, x)
    return h + 1.0 if self.training else h


def residual(self, x):
    return x + chunked(self, x)


def clamped_when_long(self, x):
    return chunked(self, x.clamp(-1, 1) if x.shape[0] > 100 else x)


def other_axis(self, x):
    gate, up = self.w12(x).chunk(2, dim=1)
    return self.w3(torch.nn.functional.silu(gate) * up)


def counting(self, x):
    self.calls = getattr(self, "calls", 0) + 1
    return chunked(self, x)


def with_a_mask(self, x, mask=None):
    return chunked(self, x if mask is None else x * mask)


def twice(self, x):
    gate, up = self.w12(x).chunk(2, dim=-1)
    torch.nn.functional.silu(gate, inplace=True)
    return self.w3(torch.nn.functional.silu(gate) * up)


def w3_only(self, x):
    return self.w3(x[..., :6])


@pytest.mark.parametrize("forward,more", [
    (gelu, {}), (up_first, {}), (scaled_and_dropped, {"scale": torch.nn.Parameter(torch.ones(6))}), (dropped, {"drop": 0.1}), (dropped, {"drop": 0.0}),
    (own_nonlinearity, {"nonlinearity": torch.nn.functional.gelu}), (own_nonlinearity, {"nonlinearity": torch.nn.GELU()}),
    (own_nonlinearity, {"nonlinearity": type("Other", (torch.nn.SiLU,), {"forward": lambda self, g: g})()}), (frozen_half, {}), (in_full_precision, {}),
    (training_noise, {}), (residual, {}), (clamped_when_long, {}), (other_axis, {}), (counting, {}), (with_a_mask, {}), (twice, {}), (w3_only, {}),
    (own_nonlinearity, {"nonlinearity": torch.nn.SiLU(inplace=True)}), (chunked, {"scale": torch.nn.Parameter(torch.ones(6))})],
    ids=lambda v: v.__name__ if callable(v) else "-".join(v))
def test_train_natively_goes_by_what_a_forward_computes(forward, more):
    """Feed-forwards that look like a gated SiLU block from outside: left alone, their results their own, nothing in them touched."""
    from iffnerf_amd import hip_vit
    m = ffn(forward, **more)
    state, x = dict(m.__dict__), torch.randn(2, 8, generator=torch.Generator().manual_seed(1))
    modes = torch.is_grad_enabled(), torch.is_autocast_enabled("cuda"), torch.get_autocast_dtype("cuda")
    torch.manual_seed(2)
    with torch.no_grad():
        want = m(x) if forward is not other_axis else None
    if forward is counting:
        del m.calls
    for training in (True, False):
        assert hip_vit.train_natively(m.train(training)) is m and m.training is training
    m.train()
    assert dict(m.__dict__).keys() == state.keys() and all(v is state[k] for k, v in m.__dict__.items())
    assert modes == (torch.is_grad_enabled(), torch.is_autocast_enabled("cuda"), torch.get_autocast_dtype("cuda"))
    torch.manual_seed(2)
    with torch.no_grad():
        assert want is None or torch.equal(m(x), want)


def sliced(self, x):
    both = self.w12(x)
    return self.w3(both[..., 6:] * torch.nn.functional.silu(both[..., :6]))


def split(self, x):
    gate, up = torch.split(self.w12(x), 6, dim=-1)
    return self.w3(torch.nn.functional.silu(gate).mul(up))


@pytest.mark.parametrize("forward,more", [(chunked, {}), (sliced, {}), (split, {}), (own_nonlinearity, {"nonlinearity": torch.nn.SiLU()}),
                                          (own_nonlinearity, {"nonlinearity": torch.nn.functional.silu}), (chunked, {"note": "w"}), (chunked, {"unused": None})])
def test_train_natively_takes_the_gated_silu_block(forward, more):
    """However it is written; and a module that is changed afterwards runs its own forward again."""
    from iffnerf_amd import hip_vit
    m, x = ffn(forward, **more), torch.randn(2, 8, generator=torch.Generator().manual_seed(1))

    def native():
        try:
            m(x)
        except RuntimeError as e:
            assert "no CPU path" in str(e)
            return True
        return False

    hip_vit.train_natively(m)
    assert "forward" in m.__dict__ and native() and not hip_vit.train_stock(m).__dict__.get("forward")
    first = hip_vit.train_natively(m).__dict__["forward"]
    assert hip_vit.train_natively(m).__dict__["forward"] is not first and native()                 # (installed again: looked at again)
    if "nonlinearity" in more:
        m.nonlinearity = torch.nn.GELU() if isinstance(more["nonlinearity"], torch.nn.Module) else torch.nn.functional.gelu
        assert not native() and torch.equal(m(x), forward(m, x))
        m.nonlinearity = more["nonlinearity"]
        assert native()
    m.act = torch.nn.functional.gelu                                          # (an attribute that a forward may look for)
    assert not native()
    del m.act
    assert native()
    m.add_module("late", torch.nn.Identity())
    assert not native()


def test_train_natively_takes_the_stand_ins_own_block():
    from iffnerf_amd import hip_vit
    from iffnerf_amd.pose_estimation.backbone import SeededViTS14
    m = hip_vit.train_natively(SeededViTS14(seed=3, dim=96, depth=2, heads=3, pretrain_grid=4, ffn="swiglu"))
    assert all(isinstance(b.mlp.__dict__["forward"], hip_vit._NativeGatedMlp) for b in m.blocks)


# ------------------------------------------------------------------------------------------------------------ forward-mode tangents
@pytest.mark.parametrize("trains", [False, True])
def test_tangents_are_refused(trains, monkeypatch):
    """Without a GPU: a dual tensor in any place that has a derivative raises, whether or not it requires a gradient, and so does a dual
    gradient; a forward-mode level alone changes nothing."""
    from torch.autograd import forward_ad
    ran = []
    monkeypatch.setattr(hip_block, "_run", lambda name, *a: ran.append(name))
    monkeypatch.setattr(hip_block, "_serves", lambda t, name: None)
    x, w, w12, b12, w3, b3 = (torch.ones(s) for s in ((3, 4), (4,), (12, 4), (12,), (4, 6), (4,)))
    for call, args in ((hip_block.layer_norm, (x, w, w)), (hip_block.gated_mlp, (x, w12, b12, w3, b3)),
                       (lambda a, r: hip_block.dropout(a, 0.5, 1, residual=r), (x, x))):
        for i in range(len(args)):
            plain = [a.clone().requires_grad_(trains) for a in args]
            with forward_ad.dual_level():
                y = call(*plain)
                assert len(ran) == 1
                dual = list(plain)
                dual[i] = forward_ad.make_dual(plain[i], torch.ones_like(plain[i]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(*dual)
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                    call(*dual)
                assert len(ran) == 1
                if trains:
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        torch.autograd.grad(y, plain, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))
                    assert len(ran) == 1
            del ran[:]
    with pytest.raises(RuntimeError):
        torch.func.jvp(hip_block.layer_norm, (x,), (x,))
    assert not ran


# ------------------------------------------------------------------------------------------------------------ what the modules around them do
@pytest.mark.parametrize("affine", [True, False])
def test_a_norm_of_another_width_is_refused(affine, monkeypatch):
    """Without a GPU: as the module's own forward refuses it, with or without parameters."""
    from iffnerf_amd import hip_vit
    ran = []
    monkeypatch.setattr(hip_block, "layer_norm", lambda x, *a: ran.append(x.shape))
    m = torch.nn.LayerNorm(8, elementwise_affine=affine)
    for x in (torch.zeros(2, 6), torch.zeros(2, 1), torch.zeros(8, 2), torch.zeros(())):
        with pytest.raises(RuntimeError):
            m(x)
        with pytest.raises(RuntimeError, match="normalized_shape"):
            hip_vit.train_natively(m)(x)
        hip_vit.train_stock(m)
    hip_vit.train_natively(m)(torch.zeros(2, 8))
    assert ran == [(2, 8)]


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("par", [torch.float32, torch.bfloat16])
def test_a_norm_under_autocast_answers_as_the_module_does(dev, dtype, par):
    """fp32 whatever comes in, gradients in the leaves' types, within the bounds of an fp32 norm of the same values; outside the region the
    input's type again."""
    from iffnerf_amd import hip_vit
    m = torch.nn.LayerNorm(40, eps=1e-6).to(dev, par)
    with torch.no_grad():
        m.weight.copy_(normal((40,), 1, par, 0.2, 1.0))
        m.bias.copy_(normal((40,), 2, par, 0.3))
    x, dy = normal((3, 7, 40), 3, dtype).requires_grad_(True), normal((3, 7, 40), 4)
    leaves = (x, m.weight, m.bias)

    def step():
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = m(x)
        return y, torch.autograd.grad(y, leaves, dy)

    stock, sgrads = step()
    hip_vit.train_natively(m)
    y, grads = step()
    assert y.dtype == stock.dtype == torch.float32 and [g.dtype for g in grads] == [g.dtype for g in sgrads]
    want, lim = norm_reference(x.detach().float(), m.weight.detach(), m.bias.detach(), 1e-6, dy)
    within(y.detach().reshape(-1, 40), want[0], lim[0], "y")
    for g, w, e, name in zip(grads, want[1:], lim[1:], ("dx", "dw", "db")):
        within(g, w, e, name)
    if par == torch.float32:
        assert m(x).dtype == dtype


@gpu
@pytest.mark.parametrize("rt", TYPES, ids=IDS)
@pytest.mark.parametrize("bt", TYPES, ids=IDS)
def test_the_sum_behind_a_dropout_is_in_the_wider_type(dev, rt, bt):
    """residual + dropout(branch) of two types, and of shapes that broadcast: the type and shape of the module's own sum, its kept positions
    to a rounding of the result, the residual exact where the branch is dropped, gradients in the leaves' types."""
    from iffnerf_amd import hip_vit
    from iffnerf_amd.pose_estimation.backbone import _DropAdd
    m = _DropAdd(0.5)
    for rs, bs in (((4, 33, 40), (4, 33, 40)), ((1, 40), (4, 33, 40)), ((4, 33, 40), (33, 40))):
        r, b = normal(rs, 5, rt).requires_grad_(True), normal(bs, 6, bt, 3.0).requires_grad_(True)
        stock = hip_vit.train_stock(m).train()(r, b)
        hip_vit.train_natively(m)
        y = m(r, b)
        assert y.dtype == stock.dtype and y.shape == stock.shape
        dy = normal(tuple(y.shape), 7, y.dtype)
        dr, db = torch.autograd.grad(y, (r, b), dy)
        assert dr.dtype == rt and db.dtype == bt and dr.shape == r.shape and db.shape == b.shape
        if rs == bs:                                           # kept: db is 2 dy, 0 where dropped
            keep = (db != 0).double()
            assert 0.4 < float(keep.mean()) < 0.6 and torch.equal(dr, dy.to(rt))
            want = r.detach().double() + 2.0 * b.detach().double() * keep
            within(y.detach(), want, 2.0 ** -23 * (want.abs() + 2.0 * b.detach().double().abs()), "y")
            assert torch.equal(y.detach()[keep == 0], r.detach().to(y.dtype)[keep == 0])


def test_a_served_backbone_in_training_mode_drops(monkeypatch):
    """serve_natively, no gradients, training mode with dropout: the module's own forward (the native one drops nothing); in evaluation and
    without a dropout the native one."""
    from iffnerf_amd import hip_vit
    from iffnerf_amd.pose_estimation.backbone import SeededViTS14
    served = []

    class Handle:
        def forward(self, x, want_cls):
            served.append(x.shape)
            return "tokens", "class"

        def close(self):
            pass

    monkeypatch.setattr(hip_vit, "ViTHandle", lambda *a, **kw: Handle())
    x = torch.randn(1, 3, 56, 56, generator=torch.Generator().manual_seed(1))

    def features(m):
        with torch.no_grad():
            return m.forward_features(x)["x_norm_patchtokens"]

    for drop, training, native in ((0.2, True, False), (0.2, False, True), (0.0, True, True)):
        m = hip_vit.serve_natively(SeededViTS14(seed=3, dim=96, depth=2, heads=3, pretrain_grid=4, drop=drop), (4, 4)).train(training)
        a, b = features(m), features(m)
        assert len(served) == 2 * native and ((a == "tokens") if native else not torch.equal(a, b))
        del served[:]


def test_a_stand_in_pickled_whole_without_its_sums_still_loads():
    """A module saved whole while its blocks had no add1 / add2: the same features after loading."""
    import pickle
    from iffnerf_amd.pose_estimation.backbone import SeededViTS14
    m = SeededViTS14(seed=3, dim=96, depth=2, heads=3, pretrain_grid=4).eval()
    x = torch.randn(1, 3, 56, 56, generator=torch.Generator().manual_seed(1))
    with torch.no_grad():
        want = m.forward_features(x)["x_prenorm"]
        for b in m.blocks:
            del b.add1, b.add2
        old = pickle.loads(pickle.dumps(m))
        assert torch.equal(old.forward_features(x)["x_prenorm"], want) and list(old.state_dict()) == list(m.state_dict())
        assert not any(k.training for k in old.modules())


# ------------------------------------------------------------------------------------------------------------ the generator, the error text
def philox(c, k):
    for _ in range(10):
        p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & 0xFFFFFFFF, (p0 >> 32) ^ c[3] ^ k[1], p0 & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def test_the_generator_gives_the_published_answers():
    """Philox 4x32-10 at all zeros, all ones and the digits of pi, and that the dropout tests' generator is the same function."""
    ones, pi = [0xFFFFFFFF] * 6, [0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344, 0xA4093822, 0x299F31D0]
    assert philox([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert philox(ones[:4], ones[4:]) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert philox(pi[:4], pi[4:]) == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]
    for seed, offset in ((0, 0), (2 ** 64 - 1, 2 ** 64 - 1), (5 << 33 | 9, 7 << 35 | 3)):
        bits = philox_bits(24, seed, offset).tolist()
        want = [w for b in range(3) for w in philox([b, 0, offset & 0xFFFFFFFF, offset >> 32], [seed & 0xFFFFFFFF, seed >> 32])]
        assert [bits[2 * i] | bits[2 * i + 1] << 16 for i in range(12)] == want


def test_the_suite_passes_in_any_order():
    """The library keeps the text of a thread's last error; a test that asks for none must not go by what another one left."""
    import os
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-p", "no:cacheprovider", "tests/test_hip_block.py::test_c_entries_refuse_bad_arguments_without_a_gpu",
                        "tests/test_abi.py::test_library_exports_every_declared_symbol"], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout[-2000:]


def test_nothing_beside_the_dma_uses_m0(tmp_path):
    """The LDS-DMA written as assembly sets m0, a register that a statement cannot name as clobbered (the compiler keeps it out of its own
    allocation and writes it right before each instruction that reads it).  In the built kernels with a k-strided operand every m0 belongs to
    that statement: set, one s_nop, the DMA."""
    import re
    import shutil
    import subprocess
    from iffnerf_amd import build
    build.build()
    shutil.copy(build.CSRC + "/block/ffn_kernels.o", tmp_path / "k.o")
    objdump = "/opt/rocm/llvm/bin/llvm-objdump"
    subprocess.run([objdump, "--offloading", "k.o"], cwd=tmp_path, check=True, capture_output=True)
    code, = tmp_path.glob("*gfx950")
    text = subprocess.run([objdump, "-d", "--no-show-raw-insn", str(code)], check=True, capture_output=True, text=True).stdout
    kernels = 0
    for body in re.split(r"^[0-9a-f]+ <", text, flags=re.M)[1:]:
        name, lines = body.split(">:", 1)
        if "k_ffn_product" not in name or not re.search(r"k_ffn_productI(f|DF16b|DF16_)Li\dELi1E", name):          # <T, AK, BK = KS, ...>
            continue
        ops = [line.split("//")[0].split() for line in lines.splitlines() if line.split("//")[0].strip()]
        uses = [i for i, op in enumerate(ops) if any("m0" == a.strip(",") for a in op[1:])]
        for i in uses:
            assert ops[i][0] == "s_mov_b32" and ops[i][1] == "m0," and ops[i + 1][0] == "s_nop" and ops[i + 2][0] == "global_load_lds_dwordx4", (name, ops[i])
        assert uses and len(uses) == sum(op[0].startswith("global_load_lds") for op in ops)
        kernels += 1
    assert kernels == 39


# ------------------------------------------------------------------------------------------------------------ infinities
INF = float("inf")


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M,D,H,O", [(1, 16, 24, 8), (3, 9, 13, 7), (8, 40, 24, 16), (12, 40, 24, 16), (70, 33, 66, 35)])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gated_mlp_infinities_are_the_formulas(dev, M, D, H, O, act, dtype):
    """An infinity in any operand, one of each sign, two that meet, one that meets a zero: every result is infinite, NaN or finite where the
    formula in 64 bits is, with and without gradients, whatever the number of rows; the finite ones are within the usual bounds."""
    places = [("x", (0, 1), INF), ("x", (M - 1, D - 1), -INF), ("w12", (2, 3), INF), ("w12", (H + 1, 0), -INF), ("w3", (1, 4), INF), ("w3", (O - 1, H - 1), -INF),
              ("b12", (5,), INF), ("b12", (H + 2,), -INF), ("b3", (3,), INF), ("dy", (0, 2), INF), ("dy", (M - 1, 1), -INF), ("dy w3", (0, 1, 4), INF),
              ("x w12", (0, 3, 2), INF), ("zero x w12", (3, 2), INF), ("zero w3 dy", (0, 1), INF), ("x", (0, 1), float("nan"))]
    for where, at, value in places:
        t = dict(zip(("x", "w12", "b12", "w3", "b3", "dy"), make_mlp(M, D, H, O, dtype, True, seed=400 + M)))
        if where == "dy w3":
            t["dy"][at[0], at[1]] = t["w3"][at[1], at[2]] = value
        elif where == "x w12":
            t["x"][at[0], at[1]] = t["w12"][at[2], at[1]] = value
        elif where == "zero x w12":
            t["x"][:, at[1]] = 0.0
            t["w12"][at[0], at[1]] = value
        elif where == "zero w3 dy":
            t["w3"][at[1]] = 0.0
            t["dy"][at] = value
        else:
            t[where][at] = value
        names = ("x", "w12", "b12", "w3", "b3")
        leaves = [t[n].requires_grad_(True) for n in names]
        y = hip_block.gated_mlp(*leaves, activation=act)
        got = (y.detach(), *torch.autograd.grad(y, leaves, t["dy"]))
        want, lim = mlp_reference(*(t[n].detach() for n in names), act, t["dy"])
        with torch.no_grad():
            got, want, lim = (*got, hip_block.gated_mlp(*leaves, activation=act)), (*want, want[0]), (*lim, lim[0])
        for g, w, e, name in zip(got, want, lim, ("y", "dx", "dw12", "db12", "dw3", "db3", "y without gradients")):
            w = w.nan_to_num(nan=float("nan"), posinf=INF, neginf=-INF)
            for kind in (torch.isnan, torch.isposinf, torch.isneginf):
                a, b = kind(g), kind(w)
                assert torch.equal(a, b), f"{value} in {where}{at}: {name}: {kind.__name__} at {a.nonzero().tolist()[:4]}, the formula at {b.nonzero().tolist()[:4]}"
            fine = w.isfinite() & e.isfinite()
            within(g[fine], w[fine], e[fine], f"{value} in {where}{at}: {name}")


class Noted(Ffn):
    forward = chunked


def test_a_trained_backbone_survives_copies_and_pickles():
    """Natively trained modules, copied and pickled: still native, on their own parameters; one pickled before forwards were looked at runs
    its own."""
    import copy
    import pickle
    from iffnerf_amd import hip_vit
    x = torch.randn(2, 8, generator=torch.Generator().manual_seed(1))
    m = hip_vit.train_natively(Noted(note="w", ratio=2.0 / 3.0, width=123456))
    for other in (copy.deepcopy(m), pickle.loads(pickle.dumps(m))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            other(x)
        assert other.__dict__["forward"].module is other
        other.ratio = 0.5
        assert torch.equal(other(x), chunked(other, x))
    old = copy.deepcopy(m)
    for name in ("children", "others", "attributes", "count"):
        del old.__dict__["forward"].__dict__[name]
    assert torch.equal(old(x), chunked(old, x))
