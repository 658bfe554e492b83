"""mpemu.functional -- operators of a language model's training step, beside the emulated cast.

    order, offsets = group_rows(expert_ids, num_experts)     # the router's tokens, expert by expert
    h = embedding(token_ids, table, scale=d ** 0.5)          # scaled lookup; the table's gradient by sorted tokens
    y = grouped_mm(x[order], w, offsets)                     # one product per expert over ragged runs of rows
    norm = clip_grad_norm_(model.parameters(), 1.0)          # one norm over all gradients, no host synchronisation

Every operator runs in hand-written gfx950 kernels (libfpemu_hip.so) on torch's current stream; tensors live on a ROCm
device, float32 / float16 / bfloat16.  Nothing here synchronises with the host: group sizes, norms and coefficients stay
on the device, so the operators (and their gradients) can be captured into a HIP graph; a capture whose leaves an eager
autograd graph still holds is refused.  Sums run in 32 bits or more and
are rounded once, in a fixed order: the same inputs give the same bits.  Derivatives are reverse mode's: a dual tensor
(torch.autograd.forward_ad) is refused with NotImplementedError.

The module forms that the quantisation hooks attach to are module_wrappers.{ScaledEmbedding, GroupedMatmul,
GroupedLinear}; the emulators clip through optimizer_step(optimizer, max_grad_norm=...).
"""
import math

import torch
from torch.autograd import Function, forward_ad
from torch.autograd.function import once_differentiable

from .pytquant.hip import _binding as _hip

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _floating(t, what, who):
    if not torch.is_tensor(t) or t.dtype not in _FLOATS:
        raise TypeError("%s: %s must be a float32, float16 or bfloat16 tensor" % (who, what))


def _integers(t, what, who):
    if not torch.is_tensor(t) or t.dtype not in (torch.int32, torch.int64):
        raise TypeError("%s: %s must be an int32 or int64 tensor" % (who, what))


def _one_device(who, *ts):
    for t in ts:
        if not t.is_cuda:
            raise RuntimeError("%s: tensors must live on a ROCm device (got %s); this build has no CPU path" % (who, t.device))
        if t.device != ts[0].device:
            raise ValueError("%s: tensors on different devices (%s, %s)" % (who, ts[0].device, t.device))


def _native():
    """The C++ front of these operators (one call with checks, allocation, launches and the autograd node), or None:
    then the same kernels are reached through ctypes."""
    return None if _hip.tracing() else _hip.ext()


def _refuse_tangents(who, *ts):
    """The kernels read addresses: a dual tensor's result would come out without its tangent."""
    for t in ts:
        if forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("%s: forward-mode derivatives are not supported (a dual tensor came in)" % who)


def _refuse_capture(who, *ts):
    """Without the native front the stream of a leaf's accumulation node is unknown, and a captured backward pass of a leaf
    that an eager graph still holds ends the process: no captured gradients there."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in ts) and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("%s: capturing a backward pass needs the native extension (_mpemu_torch.so), with tracing off" % who)


# ---- rows by group ------------------------------------------------------------------------------------------------------
def group_rows(ids, num_groups):
    """Stable order of rows by group id: (order, offsets), both int32.

    ids: integer tensor, any shape (taken flat).  order[i] is the row at place i when the rows are sorted by id, rows of
    one group in their own order; offsets has num_groups + 1 entries, group g holds places offsets[g] .. offsets[g + 1].
    Rows whose id is outside [0, num_groups) belong to no group and come last, from offsets[num_groups] on."""
    _integers(ids, "ids", "group_rows")
    _one_device("group_rows", ids)
    num_groups = int(num_groups)
    if not 1 <= num_groups <= 2 ** 31 - 2:
        raise ValueError("group_rows: num_groups must be between 1 and 2^31 - 2, got %d" % num_groups)
    ext = _native()
    if ext is not None:
        return ext.group_rows(ids, num_groups)
    ids = ids.contiguous()
    order = torch.empty(ids.numel(), dtype=torch.int32, device=ids.device)
    offsets = torch.empty(num_groups + 1, dtype=torch.int32, device=ids.device)
    return _hip.group_rows_(ids, num_groups, order, offsets)


# ---- embedding ----------------------------------------------------------------------------------------------------------
class _Embedding(Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding):
        ctx.save_for_backward(ids)
        ctx.shape, ctx.scale, ctx.padding = weight.shape, scale, padding
        out = torch.empty(tuple(ids.shape) + (weight.shape[1],), dtype=weight.dtype, device=weight.device)
        return _hip.embedding_(ids, weight.contiguous(), out, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        _refuse_tangents("embedding", grad)
        ids, = ctx.saved_tensors
        dweight = torch.empty(ctx.shape, dtype=grad.dtype, device=grad.device)
        return None, _hip.embedding_grad_(grad.contiguous(), ids, dweight, ctx.scale, ctx.padding), None, None


def _number(scale):
    """scale as a float: a tensor that autograd follows would lose its derivative here."""
    if torch.is_tensor(scale) and (scale.requires_grad or forward_ad.unpack_dual(scale).tangent is not None):
        raise TypeError("embedding: scale is a number and has no derivative; multiply the result by a scale that is learned")
    return float(scale)


def embedding(ids, weight, scale=1.0, padding_idx=None):
    """scale * weight[ids]: ids of any shape, weight [entries, width]; the result has shape ids.shape + (width,).

    The gradient of the table is dense and deterministic: tokens are sorted by entry and every entry's rows are summed in
    fp32, in token order, and rounded once.  padding_idx (negative: from the end): that entry's gradient is zero.  An id
    outside the table is not an error that the device could raise: its row of the result is NaN, it adds to no gradient.
    Differentiable once, in weight; scale is a number."""
    who = "embedding"
    _integers(ids, "ids", who)
    _floating(weight, "weight", who)
    scale = _number(scale)
    _one_device(who, ids, weight)
    if weight.dim() != 2:
        raise ValueError("embedding: weight must be 2-D, got %s" % (tuple(weight.shape),))
    if not 1 <= weight.shape[0] <= 2 ** 31 - 2:
        raise ValueError("embedding: the table needs between 1 and 2^31 - 2 entries")
    padding = -1
    if padding_idx is not None:
        padding = int(padding_idx)
        if not -weight.shape[0] <= padding < weight.shape[0]:
            raise ValueError("embedding: padding_idx %d is outside the table of %d entries" % (padding, weight.shape[0]))
        padding %= weight.shape[0]
    ext = _native()
    if ext is not None:
        return ext.embedding(ids, weight, scale, padding)
    _refuse_tangents(who, weight)
    _refuse_capture(who, weight)
    return _Embedding.apply(ids.contiguous(), weight, scale, padding)


# ---- products by group ----------------------------------------------------------------------------------------------------
def _laid_out(weight):
    """(tensor to hand to the kernel, transposed flag): a transposed view of contiguous [G, N, K] matrices -- a linear
    layer's weights -- is passed as a flag, anything else is made contiguous."""
    if weight.is_contiguous():
        return weight, False
    t = weight.transpose(1, 2)
    if t.is_contiguous():
        return t, True
    return weight.contiguous(), False


class _GroupedMm(Function):
    @staticmethod
    def forward(ctx, x, weight, offsets):
        x = x.contiguous()
        w, trans = _laid_out(weight)
        ctx.save_for_backward(x, w, offsets)
        ctx.trans = trans
        y = torch.empty((x.shape[0], weight.shape[2]), dtype=x.dtype, device=x.device)
        return _hip.grouped_gemm_(y, x, w, offsets, trans)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        _refuse_tangents("grouped_mm", grad)
        x, w, offsets = ctx.saved_tensors
        grad = grad.contiguous()
        dx = dw = None
        if ctx.needs_input_grad[0]:
            dx = _hip.grouped_gemm_(torch.empty_like(x), grad, w, offsets, not ctx.trans)
        if ctx.needs_input_grad[1]:
            dw = torch.empty_like(w)
            if ctx.trans:
                dw = _hip.grouped_gemm_wgrad_(dw, grad, x, offsets).transpose(1, 2)
            else:
                dw = _hip.grouped_gemm_wgrad_(dw, x, grad, offsets)
        return dx, dw, None


def grouped_mm(x, weight, offsets):
    """y[i] = x[i] @ weight[g] for offsets[g] <= i < offsets[g + 1]: one matrix product per group of rows.

    x [rows, K]; weight [groups, K, N] or a transposed view of [groups, N, K] (taken as it lies, no copy); offsets: int32 or
    int64, groups + 1 entries, not decreasing, as group_rows returns them.  The sizes stay on the device.  Groups may be
    empty; rows outside every group are zero in y and in the gradient of x, and add to no gradient of weight.  16-bit types
    multiply on the matrix cores with fp32 sums; fp32 runs the k-ascending fmaf chain of the c-model
    (mpemu.cmodel.simple, accumulation "fma"), whatever set_accumulation says.  Under torch.autocast x and weight are cast to
    its type first, as torch's own matrix products do.  Differentiable once, in x and weight."""
    who = "grouped_mm"
    _floating(x, "x", who)
    _floating(weight, "weight", who)
    if torch.is_autocast_enabled("cuda"):
        x, weight = (t.to(torch.get_autocast_dtype("cuda")) for t in (x, weight))
    _integers(offsets, "offsets", who)
    _one_device(who, x, weight, offsets)
    if x.dtype != weight.dtype:
        raise TypeError("grouped_mm: x is %s, weight is %s" % (x.dtype, weight.dtype))
    if x.dim() != 2 or weight.dim() != 3 or x.shape[1] != weight.shape[1] or weight.shape[0] < 1:
        raise ValueError("grouped_mm: x [rows, K] and weight [groups, K, N] expected, got %s and %s"
                         % (tuple(x.shape), tuple(weight.shape)))
    if offsets.dim() != 1 or offsets.shape[0] != weight.shape[0] + 1:
        raise ValueError("grouped_mm: offsets must have %d entries, got %s" % (weight.shape[0] + 1, tuple(offsets.shape)))
    offsets = offsets.to(torch.int32).contiguous()
    ext = _native()
    if ext is not None:
        return ext.grouped_mm(x, weight, offsets)
    _refuse_tangents(who, x, weight)
    _refuse_capture(who, x, weight)
    return _GroupedMm.apply(x, weight, offsets)


# ---- gradient norm and clipping --------------------------------------------------------------------------------------------
def _order(norm_type, who):
    order = {1.0: _hip.NORM_1, 2.0: _hip.NORM_2, math.inf: _hip.NORM_INF}.get(float(norm_type))
    if order is None:
        raise ValueError("%s: norm_type must be 1, 2 or inf, got %r" % (who, norm_type))
    return order


def _list(grads):
    return [grads] if torch.is_tensor(grads) else list(grads)


def _check_gradients(grads, who, what="a gradient"):
    for g in grads:
        if torch.is_tensor(g) and g.is_sparse:
            raise TypeError("%s: sparse gradients are not supported" % who)
        _floating(g, what, who)
        _refuse_tangents(who, g)
    _one_device(who, *grads)


def _dense(t):
    """The elements of t as one run of memory, in whatever order: t itself where it is one, else a copy."""
    t = t.detach()
    order = sorted(range(t.dim()), key=lambda i: -t.stride(i))
    return t if t.is_contiguous() or t.permute(order).is_contiguous() else t.contiguous()


def _places_meet(terms, target, most_steps=20000):
    """Whether sum(step * x) = target has a solution with 0 <= x <= most over the terms (step, most).  Strides nest in
    practice, so the search takes a few steps; one that takes more than most_steps counts as "yes"."""
    merged = {}
    for step, most in terms:
        if most > 0:
            merged[step] = merged.get(step, 0) + most
    terms = sorted(merged.items(), reverse=True)
    reach, common = [0], [0]    # of the terms from k on: their largest sum, their steps' common divisor
    for step, most in reversed(terms):
        reach.append(reach[-1] + step * most)
        common.append(math.gcd(common[-1], step))
    reach.reverse()
    common.reverse()
    todo = [(0, target)]
    while todo:
        k, t = todo.pop()
        if t < 0 or t > reach[k] or (k < len(terms) and t % common[k]):
            continue
        if k == len(terms):
            return True
        step, most = terms[k]
        lo, hi = max(0, -((reach[k + 1] - t) // step)), min(most, t // step)
        most_steps -= max(0, hi - lo + 1)
        if most_steps < 0:
            return True
        todo += [(k + 1, t - x * step) for x in range(lo, hi + 1)]
    return False


def _dims(t):
    """(stride in bytes, size) of the dimensions in which t moves, and its element size."""
    es = t.element_size()
    return [(st * es, n) for st, n in zip(t.stride(), t.shape) if n > 1], es


def _extent(t):
    """Bytes from a tensor's first to behind its last element."""
    if t.is_contiguous():
        return t.numel() * t.element_size()
    dims, es = _dims(t)
    return sum(st * (n - 1) for st, n in dims) + es


def _share_memory(a, b):
    """Whether two tensors whose extents meet have a byte in common: one linear equation in their indices (b's backwards)."""
    if a.is_contiguous() and b.is_contiguous():
        return True    # asked of extents that meet
    (da, ea), (db, eb) = _dims(a), _dims(b)
    terms = [(st, n - 1) for st, n in da + db if st > 0] + [(1, ea + eb - 2)]
    return _places_meet(terms, b.data_ptr() - a.data_ptr() + _extent(b) - 1)


def _shares_with_itself(t):
    if t.is_contiguous():
        return False
    dims, es = _dims(t)
    if any(st == 0 for st, _ in dims):
        return True
    dims.sort()
    if all(st >= sum(s * (n - 1) for s, n in dims[:k]) + es for k, (st, _) in enumerate(dims)):
        return False
    for k, (st, n) in enumerate(dims):    # two elements whose indices differ from dimension k on
        rest = dims[k + 1:]
        terms = [(st, n - 2), (1, 2 * (es - 1))] + [(s, 2 * (m - 1)) for s, m in rest]
        if _places_meet(terms, es - 1 - st + sum(s * (m - 1) for s, m in rest)):
            return True
    return False


def _overlap(grads, outs):
    """True where an output shares memory with another entry's gradient or output, or its elements with each other."""
    spans = []
    for g, o in zip(grads, outs):
        if g.numel() == 0:
            continue
        if _shares_with_itself(o):
            return True
        spans.append((o.data_ptr(), o.data_ptr() + _extent(o), True, o))
        if o.data_ptr() != g.data_ptr() or o.dtype != g.dtype:
            spans.append((g.data_ptr(), g.data_ptr() + _extent(g), False, g))
    reaching = []    # spans before this one that reach over its beginning
    for lo, hi, is_out, t in sorted(spans, key=lambda s: s[:2]):
        reaching = [r for r in reaching if r[0] > lo]
        if any((is_out or other_out) and _share_memory(other, t) for _, other_out, other in reaching):
            return True
        reaching.append((hi, is_out, t))
    return False


def _over_ranks(total, order, group):
    """The sum (or maximum) of `total` (float64[1]) over the ranks of a process group, in place.  RCCL reduces it in stream
    order; every other backend gets it staged through the host.  A NaN of one rank reaches all of them."""
    import torch.distributed as dist
    from .sharded import group_backend
    staged = total if group_backend(group) == "nccl" else total.cpu()
    if order == _hip.NORM_INF:   # a maximum need not carry a NaN: that travels beside it
        pair = torch.cat([staged.nan_to_num(nan=math.inf, posinf=math.inf), staged.isnan().to(staged.dtype)])
        dist.all_reduce(pair, op=dist.ReduceOp.MAX, group=group)
        staged = torch.where(pair[1:] > 0, math.nan, pair[:1])
    else:
        dist.all_reduce(staged, op=dist.ReduceOp.SUM, group=group)
    if staged is not total:
        total.copy_(staged)
    return total


def grad_norm(grads, norm_type=2.0):
    """The norm (1, 2 or inf) of all elements of a list of tensors as one vector: float32, 0-d, on the device.  The sum runs
    in 64 bits, so neither large nor many elements overflow or drown it (squares of 16-bit elements, exact in fp32, are
    added in fours there first wherever fp32's range holds them: two roundings of 2^-24 at most).  No derivative of the norm
    is kept."""
    who = "grad_norm"
    order = _order(norm_type, who)
    grads = _list(grads)
    if not grads:
        return torch.tensor(0.0)
    ext = _native()
    if ext is not None and all(torch.is_tensor(g) for g in grads):
        return ext.grad_norm(grads, order)
    _check_gradients(grads, who)
    dense = [_dense(g) for g in grads]
    total = torch.empty(1, dtype=torch.float64, device=grads[0].device)
    norm = torch.empty((), dtype=torch.float32, device=grads[0].device)
    _hip.grad_norm_multi_(dense, order, total, norm)
    return norm


def clip_grads_(grads, max_norm, norm_type=2.0, out=None, error_if_nonfinite=False, group=None):
    """Scale a list of gradients by min(1, max_norm / (norm + 1e-6)), norm over all of them; returns the norm (float32, 0-d,
    on the device, before clipping).

    In place, or into `out`: a list of the same shapes and strides, each of the gradient's type or float32 (16-bit model
    gradients clipped into fp32 master gradients in one pass).  No tensor may share memory with another one's output, nor
    an output's elements with each other (views that interleave are told from views that overlap).  A norm that is not
    finite gives what the arithmetic gives (NaN, or zeros and NaN), as torch.nn.utils.clip_grad_norm_ does;
    error_if_nonfinite=True reads the norm on the host first and raises instead, with every gradient as it was.

    group: a torch.distributed process group over whose ranks the gradients are sharded: the norm is that of all ranks'
    gradients (one all-reduce of one word), every rank's list on one device of its own, an empty one included."""
    who = "clip_grads_"
    order = _order(norm_type, who)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError("clip_grads_: max_norm must not be negative or NaN, got %r" % max_norm)
    grads = _list(grads)
    out = None if out is None else _list(out)
    if out is not None and len(out) != len(grads):
        raise ValueError("clip_grads_: %d gradients but %d outputs" % (len(grads), len(out)))
    if not grads and group is None:
        return torch.tensor(0.0)
    ext = _native()
    if ext is not None and group is None and all(torch.is_tensor(t) for t in grads + (out or [])):
        return ext.clip_grads(grads, out, max_norm, order, bool(error_if_nonfinite))
    _check_gradients(grads, who)
    if out is not None:
        _check_gradients(out, who, "an output")
        for g, o in zip(grads, out):
            if o.shape != g.shape or o.stride() != g.stride() or o.device != g.device or o.dtype not in (g.dtype, torch.float32):
                raise ValueError("clip_grads_: an output needs its gradient's shape, strides and device, and its type or float32")
    overlap = _overlap if _hip.ext() is None else _hip.ext().overlap
    if overlap(grads, grads if out is None else out):
        raise ValueError("clip_grads_: a gradient or output shares memory with another output (or with itself)")
    dense = [_dense(g) for g in grads]
    if out is None:
        outs = dense
    else:
        outs = [o.detach() for o in out]
        for d, g in zip(dense, grads):
            if d.data_ptr() != g.data_ptr():
                raise ValueError("clip_grads_: out needs gradients that fill their memory without gaps")
    device = grads[0].device if grads else torch.device("cuda", torch.cuda.current_device())
    total = torch.empty(1, dtype=torch.float64, device=device)
    norm = torch.empty((), dtype=torch.float32, device=device)
    _hip.grad_norm_multi_(dense, order, total)
    if group is not None:
        _over_ranks(total, order, group)
    if error_if_nonfinite:
        value = (total.sqrt() if order == _hip.NORM_2 else total).float().item()   # the norm as it is returned
        if not math.isfinite(value):
            raise RuntimeError("clip_grads_: the norm of the gradients is %s" % value)
    _hip.clip_multi_(dense, outs, order, total, max_norm, norm)
    for d, g, o in zip(dense, grads, grads if out is None else out):
        if out is None and d.data_ptr() != g.data_ptr():
            g.detach().copy_(d)
        elif not o.is_inference():
            torch.autograd.graph.increment_version(o)   # written through its address
    return norm


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False, group=None):
    """torch.nn.utils.clip_grad_norm_ on these kernels: clips the .grad of the parameters that have one, in place, and
    returns the norm before clipping.  Two passes over the gradients (one where nothing has to be clipped), a few launches
    for the whole list, no host synchronisation.  The gradients are on one device; group: as clip_grads_."""
    params = [parameters] if torch.is_tensor(parameters) else parameters
    return clip_grads_([p.grad for p in params if p.grad is not None], max_norm, norm_type, error_if_nonfinite=error_if_nonfinite,
                       group=group)
