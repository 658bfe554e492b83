"""Refusals of the training operators (mpemu.functional and their C entry points): decided on the host before anything
is enqueued, so they need no GPU."""
import ctypes

import pytest
import torch

from mpemu import functional as F
from mpemu.module_wrappers import GroupedLinear, ScaledEmbedding
from mpemu.pytquant.hip import _binding as b

INT, FLT = torch.zeros(4, dtype=torch.int64), torch.zeros(4, 4)


@pytest.mark.parametrize("call", [
    lambda: F.group_rows(INT.float(), 4), lambda: F.group_rows([1, 2], 4), lambda: F.group_rows(INT.to(torch.int16), 4),
    lambda: F.embedding(FLT, FLT), lambda: F.embedding(INT, FLT.double()), lambda: F.embedding(INT, INT),
    lambda: F.grouped_mm(INT, FLT, INT), lambda: F.grouped_mm(FLT.double(), FLT, INT),
    lambda: F.clip_grads_([INT], 1.0), lambda: F.clip_grads_([FLT.to_sparse()], 1.0), lambda: F.grad_norm([FLT.double()])])
def test_wrong_types_raise_type_error(call):
    with pytest.raises(TypeError):
        call()


@pytest.mark.parametrize("call", [
    lambda: F.group_rows(INT, 4), lambda: F.embedding(INT, FLT), lambda: F.grouped_mm(FLT, FLT[None], INT),
    lambda: F.clip_grads_([FLT], 1.0), lambda: F.grad_norm([FLT])])
def test_cpu_tensors_raise(call):
    with pytest.raises(RuntimeError, match="ROCm device"):
        call()


def test_dual_tensors_are_refused_before_anything_else():
    """A forward-mode derivative would be lost in silence: both fronts refuse the tensor that carries one."""
    from torch.autograd import forward_ad
    fronts = [b.ext()] if b.ext() is not None else []
    w3, offsets = torch.zeros(2, 4, 4), torch.tensor([0, 1, 4], dtype=torch.int32)
    with forward_ad.dual_level():
        for grad_mode in (True, False):
            with torch.set_grad_enabled(grad_mode):
                dual, dual3 = forward_ad.make_dual(FLT, torch.ones_like(FLT)), forward_ad.make_dual(w3, torch.ones_like(w3))
                calls = [lambda: F._refuse_tangents("x", FLT, dual), lambda: F._check_gradients([FLT, dual], "x")]
                for e in fronts:
                    calls += [lambda: e.embedding(INT, dual, 1.0, -1), lambda: e.grouped_mm(dual, w3, offsets),
                              lambda: e.grouped_mm(FLT, dual3, offsets), lambda: e.grouped_mm(FLT, dual3.transpose(1, 2), offsets),
                              lambda: e.grad_norm([dual], b.NORM_2), lambda: e.clip_grads([FLT, dual], None, 1.0, b.NORM_2, False)]
                for call in calls:
                    with pytest.raises(NotImplementedError, match="forward-mode"):
                        call()
        F._refuse_tangents("x", FLT)


def test_a_scale_to_learn_is_refused():
    from torch.autograd import forward_ad
    learned = torch.nn.Parameter(torch.tensor(2.0))
    for call in (lambda: F.embedding(INT, FLT, scale=learned), lambda: ScaledEmbedding(4, 4, scale=learned)):
        with pytest.raises(TypeError, match="scale"):
            call()
    with forward_ad.dual_level(), pytest.raises(TypeError, match="scale"):
        F.embedding(INT, FLT, scale=forward_ad.make_dual(torch.tensor(2.0), torch.tensor(1.0)))
    assert ScaledEmbedding(4, 4, scale=torch.tensor(2.0)).scale == ScaledEmbedding(4, 4, scale=2).scale == 2.0


def test_values_refused_without_gpu():
    with pytest.raises(ValueError):
        F.grad_norm([], norm_type=3.0)
    with pytest.raises(ValueError):
        F.clip_grads_([], -1.0)
    with pytest.raises(ValueError):
        F.clip_grads_([], float("nan"))
    assert float(F.grad_norm([])) == 0.0
    assert float(F.clip_grad_norm_([torch.nn.Parameter(FLT)], 1.0)) == 0.0    # no gradient yet


def test_overlap_rule():
    t = torch.zeros(64)
    a, c = t[:16], t[16:32]
    assert not F._overlap([a, c], [a, c])                 # in place, side by side
    assert F._overlap([a, a], [a, a])                     # the same buffer twice
    assert F._overlap([t[:17], c], [t[:17], c])
    assert not F._overlap([a, a], [t[32:48], t[48:]])     # read twice, written apart
    assert F._overlap([a, c], [c, t[32:48]])              # an output is another one's gradient
    assert not F._overlap([t[:0], t[:0]], [t[:0], t[:0]])


def _bytes(t):
    """The address of every byte of t, with repetitions."""
    places = [t.data_ptr()]
    for st, n in zip(t.stride(), t.shape):
        places = [p + st * t.element_size() * i for p in places for i in range(n)]
    return [p + k for p in places for k in range(t.element_size())]


def _overlap_by_enumeration(grads, outs):
    taken = {}
    for i, (g, o) in enumerate(zip(grads, outs)):
        own = _bytes(o)
        if len(set(own)) < len(own):
            return True
        for p in own:
            if p in taken:
                return True
            taken[p] = i
    for g, o in zip(grads, outs):
        if g.data_ptr() == o.data_ptr() and g.dtype == o.dtype:
            continue
        if any(p in taken for p in _bytes(g)):
            return True
    return False


OVERLAPS = [F._overlap] + ([b.ext().overlap] if b.ext() is not None else [])


@pytest.mark.parametrize("overlap", OVERLAPS)
def test_overlap_of_tensors_with_gaps(overlap):
    s = torch.zeros(40, 30)
    shared = [[s[:, ::2], s[:, ::2]], [s[:, ::2], s], [s[::2], s[:, ::2]], [s[:, :11], s[:, 10:]], [s[:, :20:3], s.t()[3:]],
              [torch.zeros(64).as_strided((4, 4), (2, 1))], [torch.zeros(64).as_strided((3, 4), (1, 2))], [s[:1].expand(9, 30)],
              [s[3], s[:, 7]]]
    apart = [[s[:, ::2], s[:, 1::2]], [s[:, :10], s[:, 10:]], list(s.unbind(1)), [s[::2], s[1::2, ::2], s[1::2, 1::2]],
             [torch.zeros(64).as_strided((2, 3), (3, 2))], [s.t()], [s[:, None, ::3], s[:, 1::3], s.t()[2::3]], [s[:0], s]]
    for want, lists in ((True, shared), (False, apart)):
        for ts in lists:
            assert _overlap_by_enumeration(ts, ts) == want
            assert overlap(ts, ts) == want
    wide = torch.zeros(1 << 20).as_strided((1 << 9, 1 << 9), (1 << 11, 2))    # no search over elements
    assert overlap([wide, wide.t()], [wide, wide.t()]) and not overlap([wide], [wide])


@pytest.mark.parametrize("overlap", OVERLAPS)
def test_overlap_rule_on_random_views(overlap):
    """Against the addresses of every byte: views of any strides, types mixed, in place and into other views."""
    import random
    rng = random.Random(5)
    pool = torch.zeros(4096, dtype=torch.uint8)
    seen = [0, 0]

    def view(dtype=None, like=None):
        dtype = dtype or rng.choice([torch.float32, torch.float16])
        es = torch.empty(0, dtype=dtype).element_size()
        base = pool[rng.randrange(0, 300) * es:]
        base = base[:base.numel() // es * es].view(dtype)
        if like is not None:
            return base.as_strided(like.shape, like.stride())
        shape = [rng.choice([1, 2, 3, 5]) for _ in range(rng.randint(0, 3))]
        return base.as_strided(shape, [rng.choice([1, 2, 3, 4, 6, 10, 12, 30]) for _ in shape])

    for _ in range(1500):
        grads = [view() for _ in range(rng.randint(1, 3))]
        outs = grads if rng.random() < 0.6 else [view(rng.choice([g.dtype, torch.float32]), g) for g in grads]
        want = _overlap_by_enumeration(grads, outs)
        seen[want] += 1
        assert overlap(grads, outs) == want, [(t.shape, t.stride(), t.data_ptr() - pool.data_ptr()) for t in grads + outs]
    assert min(seen) > 200


def test_dense_views():
    w = torch.zeros(8, 6, 3, 3).contiguous(memory_format=torch.channels_last)
    assert F._dense(w).data_ptr() == w.data_ptr() and F._dense(w.t() if w.dim() == 2 else w).data_ptr() == w.data_ptr()
    assert F._dense(torch.zeros(4, 6)[:, ::2]).data_ptr() != 0 and F._dense(torch.zeros(4, 6)[:, ::2]).is_contiguous()


def test_c_entries_refuse():
    L = b.lib()
    # ids: null, odd sizes, too many rows or groups, misaligned
    assert L.fpemu_group_rows(None, 8, 4, 4, 16, 16, None, 0, None) == -1
    assert L.fpemu_group_rows(16, 2, 4, 4, 16, 16, None, 0, None) == -1
    assert L.fpemu_group_rows(16, 8, 1 << 31, 4, 16, 16, None, 0, None) == -1
    assert L.fpemu_group_rows(16, 8, 4, 0, 16, 16, None, 0, None) == -1
    assert L.fpemu_group_rows(16, 8, 4, (1 << 31) - 1, 16, 16, None, 0, None) == -1
    assert L.fpemu_group_rows(20, 8, 4, 4, 16, 16, None, 0, None) == -4
    assert L.fpemu_group_rows(16, 8, 4, 4, 16, None, None, 0, None) == -1
    assert L.fpemu_group_rows(16, 8, 8192, 4, 16, 16, None, 0, None) == -1            # workspace missing
    assert L.fpemu_group_rows(16, 8, 8192, 4, 16, 16, 16, 64, None) == -1             # workspace too small
    assert L.fpemu_group_rows_workspace_bytes(8192, 4) > 64
    # embedding
    assert L.fpemu_embedding(16, 16, 8, 16, 4, 8, 8, 3, 1.0, None) == -1              # fp64
    assert L.fpemu_embedding(None, 16, 8, 16, 4, 8, 8, 0, 1.0, None) == -1
    assert L.fpemu_embedding(18, 16, 8, 16, 4, 8, 8, 0, 1.0, None) == -4
    assert L.fpemu_embedding(16, 16, 8, 16, 0, 8, 8, 0, 1.0, None) == 0               # nothing to do
    assert L.fpemu_embedding(16, 16, 8, 16, 4, 8, 0, 0, 1.0, None) == 0
    assert L.fpemu_embedding_grad(16, 16, 8, 16, 4, 8, 8, 0, 1.0, -1, None, 0, None) == -1
    assert L.fpemu_embedding_grad(16, 16, 8, 16, 4, 8, 8, 0, 1.0, -1, 16, 8, None) == -1
    # grouped products
    assert L.fpemu_grouped_gemm(16, 16, 16, None, 4, 4, 4, 2, 0, 0, None) == -1
    assert L.fpemu_grouped_gemm(16, 16, 16, 16, 4, 4, 4, 0, 0, 0, None) == -1
    assert L.fpemu_grouped_gemm(16, 16, 16, 16, -1, 4, 4, 2, 0, 0, None) == -1
    assert L.fpemu_grouped_gemm(16, 16, 16, 16, 4, 4, 4, 2, 3, 0, None) == -1
    assert L.fpemu_grouped_gemm(None, 16, 16, 16, 4, 4, 4, 2, 0, 0, None) == -1
    assert L.fpemu_grouped_gemm(18, 16, 16, 16, 4, 4, 4, 2, 0, 0, None) == -4
    assert L.fpemu_grouped_gemm(16, 16, 16, 16, 0, 4, 4, 2, 0, 0, None) == 0
    assert L.fpemu_grouped_gemm_wgrad(16, 16, 16, 16, 4, 0, 4, 2, 0, None) == 0
    assert L.fpemu_grouped_gemm_wgrad(None, 16, 16, 16, 4, 4, 4, 2, 0, None) == -1
    # norm and clipping
    tab = (b._GradEntry * 2)()
    tab[0].inp, tab[0].out, tab[0].n, tab[0].in_dtype, tab[0].out_dtype = 4096, 4096, 4, 0, 0
    tp = ctypes.cast(tab, ctypes.c_void_p)
    assert L.fpemu_grad_norm_multi(tp, 1, 7, 16, None, 16, 1 << 20, None) == -1       # order
    assert L.fpemu_grad_norm_multi(tp, 1, 2, None, None, 16, 1 << 20, None) == -1
    assert L.fpemu_grad_norm_multi(tp, 1, 2, 16, None, 16, 8, None) == -1             # workspace too small
    assert L.fpemu_grad_norm_multi(None, 1, 2, 16, None, 16, 1 << 20, None) == -1
    assert L.fpemu_clip_multi(tp, 1, 2, 16, -1.0, None, None) == -1
    assert L.fpemu_clip_multi(tp, 1, 2, 16, float("nan"), None, None) == -1
    assert L.fpemu_clip_multi(tp, 1, 2, None, 1.0, None, None) == -1
    tab[0].out = 4104                                                                 # overlaps its gradient
    assert L.fpemu_clip_multi(tp, 1, 2, 16, 1.0, None, None) == -1
    assert b"overlap" in L.fpemu_last_error()
    tab[0].out, tab[0].out_dtype = 8192, 1                                            # fp32 into fp16
    assert L.fpemu_clip_multi(tp, 1, 2, 16, 1.0, None, None) == -1
    tab[0].inp = 4098
    assert L.fpemu_clip_multi(tp, 1, 2, 16, 1.0, None, None) == -4


def test_modules_and_their_hooks_configure():
    """The wrappers are hook targets: experts and embeddings get the configurations of linear layers and embeddings."""
    from mpemu.e4m3_emu import E4M3Emulator
    from mpemu.hybrid_emu import HybridEmulator
    from mpemu.module_wrappers import GroupedMatmul

    class Model(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.emb = ScaledEmbedding(10, 8, padding_idx=1, scale=2.0)
            self.experts = GroupedLinear(3, 8, 4)
            self.product = GroupedMatmul()
            self.lin = torch.nn.Linear(8, 4)

    model = Model().train()
    assert "scale=2.0" in repr(model.emb) and "num_groups=3" in repr(model.experts)
    assert float(model.emb.weight.detach()[1].abs().sum()) == 0.0          # nn.Embedding's own rule for the padding entry
    emu = HybridEmulator(model, None, device="cpu")
    emu.prepare_model(model, None, None)
    d = emu.model_qconfig_dict
    assert repr(d["experts"]) == repr(d["lin"])
    assert d["emb"].iact_qconfig is None and d["product"].wt_qconfig is None
    assert model.experts.weight._backward_hooks            # weight gradients are quantised, as a linear layer's
    emu = E4M3Emulator(Model(), None, device="cpu", train=True)
    emu.prepare_model(emu.model, None, None)
    assert emu.model_qconfig_dict["experts"].wt_qconfig is not None
    assert emu.model_qconfig_dict["product"].wt_qconfig is None


def _ranks(rank, world, path, values, out):
    import torch.distributed as dist
    dist.init_process_group("gloo", init_method="file://" + path, rank=rank, world_size=world)
    got = []
    for order, per_rank in values:
        total = torch.tensor([per_rank[rank]], dtype=torch.float64)
        got.append(float(F._over_ranks(total, order, dist.group.WORLD)))
    torch.save(got, "%s.%d" % (out, rank))
    dist.destroy_process_group()


def test_norm_over_two_ranks(tmp_path):
    """The word that ranks exchange: sums add up, maxima win, a NaN or infinity of one rank reaches the other."""
    import math
    inf, nan = math.inf, math.nan
    values = [(b.NORM_2, (2.0, 3.5)), (b.NORM_1, (0.0, 1.25)), (b.NORM_INF, (2.0, 3.5)), (b.NORM_INF, (7.0, 0.0)),
              (b.NORM_INF, (nan, 3.0)), (b.NORM_INF, (inf, nan)), (b.NORM_INF, (inf, 1.0)), (b.NORM_2, (nan, 1.0))]
    torch.multiprocessing.spawn(_ranks, args=(2, str(tmp_path / "store"), values, str(tmp_path / "out")), nprocs=2)
    want = [5.5, 1.25, 3.5, 7.0, nan, nan, inf, nan]
    for rank in range(2):
        got = torch.load(str(tmp_path / "out") + ".%d" % rank)
        assert all(g == w or (math.isnan(g) and math.isnan(w)) for g, w in zip(got, want)), got
