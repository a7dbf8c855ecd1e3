"""Class-score operators without a GPU: refusals of the public entry points and of the C ABI (before any launch), row layouts."""
import ctypes
import re

import pytest
import torch

NAN = float("nan")


@pytest.fixture(scope="module")
def log_probs():
    from vitm_amd import log_probs
    return log_probs


@pytest.fixture(scope="module")
def DistillationLoss():
    from vitm_amd.training import DistillationLoss
    return DistillationLoss


@pytest.mark.parametrize("kw,exc,words", [
    (dict(logits=torch.zeros(3, 5, dtype=torch.float16)), TypeError, "float16"),
    (dict(logits=torch.zeros(3, 5, dtype=torch.int64)), TypeError, "int64"),
    (dict(logits=torch.tensor(1.0)), ValueError, "class dimension"),
    (dict(logits=torch.zeros(3, 0)), ValueError, "0 classes"),
    (dict(logits=torch.zeros(1, 500001)), ValueError, "500001 classes"),
    (dict(logits=torch.zeros(3, 5), top_k=6), ValueError, "top_k 6"),
    (dict(logits=torch.zeros(3, 500), top_k=129), ValueError, "top_k 129"),
    (dict(logits=torch.zeros(3, 5), top_k=-1), ValueError, "top_k -1"),
    (dict(logits=torch.zeros(3, 5), temperature=0.0), ValueError, "temperature"),
    (dict(logits=torch.zeros(3, 5), temperature=-1.0), ValueError, "temperature"),
    (dict(logits=torch.zeros(3, 5), temperature=NAN), ValueError, "temperature"),
    (dict(logits=torch.zeros(3, 5), temperature=float("inf")), ValueError, "temperature"),
    (dict(logits=torch.zeros(3, 5), temperature=1e-7), ValueError, "temperature"),
    (dict(logits=torch.zeros(3, 5), temperature=2e6), ValueError, "temperature"),
    (dict(logits=torch.zeros(3, 5), targets=torch.zeros(4, dtype=torch.int64)), ValueError, "targets of shape"),
    (dict(logits=torch.zeros(3, 5), targets=torch.zeros(3)), TypeError, "int64 or int32"),
    (dict(logits=torch.zeros(3, 5), targets=torch.zeros(3, 129, dtype=torch.int64)), ValueError, "129 targets"),
    (dict(logits=torch.zeros(3, 5), targets=torch.zeros(3, dtype=torch.int64, device="meta")), RuntimeError, "meta"),
    (dict(logits=torch.zeros(3, 5)), RuntimeError, "MI355X"),
])
def test_log_probs_refuses(log_probs, kw, exc, words):
    with pytest.raises(exc, match=words):
        log_probs(kw.pop("logits"), kw.pop("targets", None), **kw)


def _args(R=3, V=9, K=4, **over):
    d = dict(logits=torch.zeros(R, V), teacher_logprobs=torch.zeros(R, K), teacher_indices=torch.zeros(R, K, dtype=torch.int64),
             labels=None)
    d.update(over)
    return d


@pytest.mark.parametrize("init,over,exc,words", [
    (dict(label_weight=1.5), None, ValueError, "label_weight"),
    (dict(label_weight=-0.1), None, ValueError, "label_weight"),
    (dict(temperature=0.0), None, ValueError, "temperature"),
    (dict(temperature=NAN), None, ValueError, "temperature"),
    (dict(reduction="median"), None, ValueError, "median"),
    (dict(), dict(logits=torch.zeros(3, 9, dtype=torch.float16)), TypeError, "float16"),
    (dict(), dict(teacher_logprobs=torch.zeros(2, 4)), ValueError, "teacher log probabilities"),
    (dict(), dict(teacher_logprobs=torch.zeros(3, 0), teacher_indices=torch.zeros(3, 0, dtype=torch.int64)), ValueError, "1 to 128"),
    (dict(), dict(teacher_logprobs=torch.zeros(3, 129), teacher_indices=torch.zeros(3, 129, dtype=torch.int64)), ValueError, "1 to 128"),
    (dict(), dict(teacher_indices=torch.zeros(3, 5, dtype=torch.int64)), ValueError, "indices of shape"),
    (dict(), dict(teacher_indices=torch.zeros(3, 4)), TypeError, "int64 or int32"),
    (dict(), dict(teacher_logprobs=torch.zeros(3, 4, dtype=torch.float64)), TypeError, "float64"),
    (dict(), dict(teacher_logprobs=torch.zeros(3, 4, requires_grad=True)), ValueError, "detach"),
    (dict(), dict(teacher_logprobs=torch.zeros(3, 4, device="meta")), RuntimeError, "meta"),
    (dict(label_weight=0.5), dict(), ValueError, "needs labels"),
    (dict(), dict(labels=torch.zeros(4, dtype=torch.int64)), ValueError, "labels of shape"),
    (dict(), dict(labels=torch.zeros(3)), TypeError, "int64 or int32"),
    (dict(), dict(), RuntimeError, "MI355X"),
])
def test_distillation_refuses(DistillationLoss, init, over, exc, words):
    with pytest.raises(exc, match=words):
        loss = DistillationLoss(**init)
        loss(**_args(**over))
    if over is not None and words != "detach":       # loss_and_grad records no graph: nothing to detach from
        with pytest.raises(exc, match=words):
            DistillationLoss(**init).loss_and_grad(**_args(**over))


def test_trainer_refuses_what_it_cannot_distil():
    from vitm_amd import training
    lin = torch.nn.Linear(2, 2)
    with pytest.raises(ValueError, match="reduction"):
        training.Trainer(lin, None, distillation=training.DistillationLoss(reduction="none"))
    with pytest.raises(ValueError, match="needs a distillation loss"):
        training.Trainer(lin, None, teacher=lin)
    with pytest.raises(ValueError, match="teacher_top_k"):
        training.Trainer(lin, None, distillation=training.DistillationLoss(), teacher_top_k=0)


@pytest.mark.parametrize("make,copies", [
    (lambda: torch.randn(7, 10), False),
    (lambda: torch.randn(7, 16)[:, 3:13], False),
    (lambda: torch.randn(4, 6, 10)[:, :-1], False),
    (lambda: torch.randn(4, 6, 16)[:, 1:, 2:12], False),
    (lambda: torch.randn(1, 10).expand(5, 10), False),
    (lambda: torch.randn(10), False),
    (lambda: torch.randn(3, 1, 5, 1, 10), False),
    (lambda: torch.randn(2, 3, 4, 10)[:, :2, :3], True),
    (lambda: torch.randn(10, 7).t(), True),
    (lambda: torch.randn(6, 20)[:, ::2], True),
    (lambda: torch.randn(8, 10)[::2], False),
    (lambda: torch.randn(5, 4, 10).transpose(0, 1), False),
    (lambda: torch.randn(9, 1), False),
    (lambda: torch.randn(9, 4)[:, :1], False),
])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_address_the_tensor(make, copies, dtype):
    """Every row at the address the layout gives holds the row of the tensor; the gradient's rows start at the same place of a
    16-byte granule."""
    from vitm_amd import _score_ops as S
    x = make().to(dtype) if make().is_contiguous() else make()
    if x.dtype != dtype:
        base = x._base.to(dtype)
        x = base.as_strided(x.shape, x.stride(), x.storage_offset())
    r = S.rows_of(x)
    assert (r.t.data_ptr() != x.data_ptr()) == copies
    flat = x.reshape(-1, x.shape[-1])
    assert (r.R, r.V) == tuple(flat.shape)
    mem = torch.as_strided(r.t, (r.t.untyped_storage().nbytes() // r.t.element_size(),), (1,), 0)
    first = r.t.storage_offset()
    dz, ld_outer, ld = S.empty_rows_like(r, x.shape)
    assert dz.shape == x.shape and dz.dtype == x.dtype
    out = torch.as_strided(dz, (dz.untyped_storage().nbytes() // dz.element_size(),), (1,), 0)
    at = lambda i, lo, l: (i // r.inner) * lo + (i % r.inner) * l
    spans = []
    for i in range(r.R):
        a = first + at(i, r.ld_outer, r.ld)
        assert torch.equal(mem[a:a + r.V], flat[i])
        b = dz.storage_offset() + at(i, ld_outer, ld)
        spans.append(b)
        assert b + r.V <= out.numel()
        assert (r.t.data_ptr() - first * r.t.element_size() + a * r.t.element_size()) % 16 == (out.data_ptr() + b * dz.element_size()) % 16
        out[b:b + r.V] = i
    assert torch.equal(dz.reshape(-1, r.V)[:, 0].float(), torch.arange(r.R).to(dtype).float())
    assert sorted(spans) == spans and all(y - x >= r.V for x, y in zip(spans, spans[1:]))


def test_c_abi_refuses_before_any_launch():
    """A host buffer stands in for device memory: only addresses are looked at."""
    from vitm_amd import _lib
    lib = _lib.load()
    buf = ctypes.create_string_buffer(8192)
    p = ctypes.c_void_p((ctypes.addressof(buf) + 255) & ~255)
    odd = ctypes.c_void_p(((ctypes.addressof(buf) + 255) & ~255) + 1)
    f = ctypes.c_float

    def lp(logits=p, dtype=1, ld=9, inner=3, R=3, V=9, T=1.0, targets=p, G=1, K=0, out=p, top=p):
        return lib.vitm_log_probs(logits, dtype, 0, ld, inner, R, V, f(T), targets, G, -100, K, out, p, p, top, top, p, None)

    def refused(rc, words):
        assert rc == -1 and re.search(words, lib.vitm_last_error().decode()), lib.vitm_last_error()

    refused(lp(logits=None), "null")
    refused(lp(dtype=7), "dtype 7")
    refused(lp(R=0), "number of rows")
    refused(lp(inner=0), "number of rows")
    refused(lp(V=0), "0 classes")
    refused(lp(V=500001), "classes")
    refused(lp(ld=-1), "stride")
    refused(lp(logits=odd), "aligned")
    refused(lp(T=0.0), "temperature")
    refused(lp(T=NAN), "temperature")
    refused(lp(T=1e-7), "temperature")
    refused(lp(R=1 << 26, inner=1 << 26), "exceed one launch")
    refused(lp(targets=None), "null")
    refused(lp(G=129), "129 targets")
    refused(lp(K=10), "top_k 10")
    refused(lp(K=129, V=500), "top_k 129")
    refused(lp(K=2, top=None), "null")
    def lpb(stats=p, targets=p, top=p, ent=p, dz=p, ldd=9, g=p, gt=p, ge=p, G=1, K=2):
        return lib.vitm_log_probs_bwd(p, 1, 0, 9, 3, 3, 9, f(1.0), targets, G, -100, top, K, stats, ent, g, p, ge, gt, dz, 0, ldd, None)

    refused(lpb(stats=None), "null")
    refused(lpb(targets=None), "null")
    refused(lpb(top=None), "null")
    refused(lpb(ent=None), "null")
    refused(lpb(dz=None), "null")
    refused(lpb(ldd=8), "overlap")
    refused(lpb(G=129), "129 targets")
    refused(lpb(), "same memory")

    def ds(T=1.0, a=0.0, tl=p, idx=p, K=4, labels=p, red=1, rl=p, loss=p, inv=p, state=p, dz=None, ldd=9, V=9, R=3):
        return lib.vitm_distill(p, 1, 0, V, R, R, V, f(T), f(a), 0, tl, idx, K, labels, -100, red, rl, loss, inv, state, dz, 0, ldd,
                                None)

    refused(ds(T=-1.0), "temperature")
    refused(ds(a=1.5), "label weight")
    refused(ds(a=0.5, labels=None), "needs labels")
    refused(ds(tl=None), "null")
    refused(ds(idx=None), "null")
    refused(ds(K=0), "list of 0")
    refused(ds(K=129), "list of 129")
    refused(ds(red=3), "reduction 3")
    refused(ds(rl=None), "null")
    refused(ds(loss=None), "null")
    refused(ds(inv=None), "inv_count")
    refused(ds(dz=p, ldd=5), "overlap")
    refused(ds(dz=p), "same memory")
    refused(ds(V=500001), "classes")
    bwd = lambda state=p, up=p, inv=p, red=1: lib.vitm_distill_bwd(p, 1, 0, 9, 3, 3, 9, f(1.0), f(0.0), 0, p, p, 4, p, -100, red, inv, state,
                                                                   up, p, 0, 9, None)
    refused(bwd(state=None), "null")
    refused(bwd(up=None), "null")
    refused(bwd(inv=None), "inv_count")
    refused(bwd(red=5), "reduction 5")
    refused(bwd(), "same memory")


def test_constants_of_the_binding():
    from vitm_amd import _lib
    lib = _lib.load()
    assert (_lib.SCORES_MAX_CLASSES, _lib.SCORES_MAX_TOP, _lib.DISTILL_STATE) == (
        lib.vitm_scores_max_classes(), lib.vitm_scores_max_top(), lib.vitm_distill_state_floats())


def test_oracle_gradients_are_differences():
    """The formulas of the 64-bit oracle against central differences of its own values."""
    import score_oracle as O
    g = torch.Generator().manual_seed(3)
    z = torch.randn(3, 8, generator=g, dtype=torch.float64)
    tgt = torch.tensor([[1, 1], [7, -100], [0, 3]])
    gl, ge, gs = torch.randn(3, 2, generator=g), torch.randn(3, generator=g), torch.randn(3, generator=g)
    T = 1.7
    value = lambda z: (lambda o: (o["logprobs"] * gl).sum() + (o["entropy"] * ge).sum() + (o["lse"] * gs).sum())(O.log_probs(z, tgt, 2, T))
    got, _ = O.log_probs_grad(O.log_probs(z, tgt, 2, T), tgt, T, gl, gs, ge)
    idx = torch.tensor([[2, 5, 2], [1, -1, 6], [0, 1, 2]])
    tl = torch.log_softmax(torch.randn(3, 4, generator=g, dtype=torch.float64), 1)[:, :3]
    lab = torch.tensor([2, -100, 7])

    def diff(fn):
        d = torch.zeros_like(z)
        for i in range(z.numel()):
            e = torch.zeros_like(z).view(-1)
            e[i] = 1e-5
            d.view(-1)[i] = (fn(z + e.view_as(z)) - fn(z - e.view_as(z))) / 2e-5
        return d

    assert (got - diff(value)).abs().max() < 1e-8
    for tail in (False, True):
        for a in (0.0, 0.4, 1.0):
            _, _, dz, _ = O.distill(z, tl, idx, lab, T, a, tail)
            d = diff(lambda z: O.distill(z, tl, idx, lab, T, a, tail)[0].sum())
            assert (dz - d).abs().max() < 1e-8, (tail, a)


def test_c_abi_refuses_a_gradient_that_meets_the_logits():
    """Shifted by a class, from in front or behind, or with another pitch, not only at the same address; rows that lie next to the
    others, as in an interleaved buffer, are not a meeting (test_gpu_scores.py runs them)."""
    from vitm_amd import _lib
    lib = _lib.load()
    buf = ctypes.create_string_buffer(1 << 16)
    at = lambda floats: ctypes.c_void_p(((ctypes.addressof(buf) + 255) & ~255) + 4 * floats)
    p, f, V, R = at(8192), ctypes.c_float, 9, 6

    def all_refuse(z, ld_outer, ld, inner, dz, ldd_outer, ldd):
        rows = (z, 1, ld_outer, ld, inner, R, V, f(1.0))
        for call, args in ((lib.vitm_log_probs_bwd, (p, 1, -100, p, 2, p, p, p, p, p, p)),
                           (lib.vitm_distill, (f(0.0), 0, p, p, 4, p, -100, 1, p, p, p, p)),
                           (lib.vitm_distill_bwd, (f(0.0), 0, p, p, 4, p, -100, 1, p, p, p))):
            rc = call(*rows, *args, dz, ldd_outer, ldd, None)
            assert rc == -1 and b"same memory" in lib.vitm_last_error(), (rc, lib.vitm_last_error())

    all_refuse(at(0), 0, 9, R, at(1), 0, 9)
    all_refuse(at(53), 0, 9, R, at(0), 0, 9)           # the last class of the last row
    all_refuse(at(0), 0, 20, R, at(8), 0, 20)
    all_refuse(at(12), 0, 20, R, at(0), 0, 20)         # the end of a row in the next one's start
    all_refuse(at(0), 0, 0, R, at(4), 0, 9)            # one row of logits, repeated
    all_refuse(at(0), 100, 10, 3, at(35), 60, 11)      # two strides
    all_refuse(at(85), 9, 1, 3, at(0), 60, 11)


def test_more_rows_than_the_c_abi_counts_are_refused(log_probs, DistillationLoss):
    """2^32 + 5 rows would arrive as 5."""
    z = torch.zeros(1, 2).expand(2 ** 32 + 5, 2)
    with pytest.raises(ValueError, match="4294967301 rows"):
        log_probs(z)
    each = lambda t: t.expand(2 ** 32 + 5, 1)
    with pytest.raises(ValueError, match="4294967301 rows"):
        DistillationLoss()(z, each(torch.zeros(1, 1)), each(torch.zeros(1, 1, dtype=torch.int64)))
    with pytest.raises(RuntimeError, match="MI355X"):
        log_probs(torch.zeros(1, 2).expand(2 ** 30, 2))


def test_rows_beyond_one_launch_are_refused_by_what_is_launched():
    """fewer than 2^32 threads: 2^22 rows of 1024 threads are too many, 2^22 rows of 64 are not (test_gpu_scores.py runs more)."""
    from vitm_amd import _lib
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.c_void_p((ctypes.addressof(buf) + 255) & ~255)
    f = ctypes.c_float

    def refused(rc):
        assert rc == -1 and b"exceed one launch" in lib.vitm_last_error(), (rc, lib.vitm_last_error())

    R, V = 1 << 22, 300000                        # a row of more than 32768 granules; every row the same one
    refused(lib.vitm_log_probs(p, _lib.BF16, 0, 0, R, R, V, f(1.0), p, 1, -100, 2, p, p, p, p, p, p, None))
    R = 1 << 24                                   # 256 threads a row
    refused(lib.vitm_log_probs(p, _lib.BF16, 0, 0, R, R, 5000, f(1.0), p, 1, -100, 2, p, p, p, p, p, p, None))
    refused(lib.vitm_distill(p, _lib.BF16, 0, 0, R, R, 5000, f(1.0), f(0.0), 0, p, p, 4, None, -100, 2, p, p, p, p, None, 0, 0, None))
    R = 1 << 26                                   # 64
    refused(lib.vitm_log_probs(p, _lib.BF16, 0, 0, R, R, 8, f(1.0), p, 1, -100, 2, p, p, p, p, p, p, None))


def test_forward_mode_is_refused(log_probs, DistillationLoss):
    """A dual tensor asks for no gradient, so its tangent would be left out in silence."""
    from torch.autograd import forward_ad as fw
    z, tl, idx = torch.zeros(3, 9), torch.zeros(3, 4), torch.zeros(3, 4, dtype=torch.int64)
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))
        for f in (lambda: log_probs(dual(z)), lambda: log_probs(dual(z[:0])), lambda: DistillationLoss()(dual(z), tl, idx),
                  lambda: DistillationLoss().loss_and_grad(dual(z), tl, idx), lambda: DistillationLoss()(z, dual(tl), idx),
                  lambda: DistillationLoss().loss_and_grad(z, dual(tl), idx)):
            with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
                f()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="no forward-mode derivative"):
                f()
        with pytest.raises(RuntimeError, match="MI355X"):
            log_probs(z)                          # a plain tensor inside a dual level


def test_temperatures_of_distillation(DistillationLoss):
    """Beyond 1e4 the gradient would have no digit left; log_probs has no such differences."""
    with pytest.raises(ValueError, match="1e-6 to 10000"):
        DistillationLoss(temperature=2e4)
    loss = DistillationLoss(temperature=1e4)
    loss.temperature = 2e4
    with pytest.raises(ValueError, match="1e-6 to 10000"):
        loss(**_args())
    from vitm_amd import _lib
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096)
    p, f = ctypes.c_void_p((ctypes.addressof(buf) + 255) & ~255), ctypes.c_float
    rows = (p, 1, 0, 9, 3, 3, 9, f(2e4), f(0.0), 0, p, p, 4, None, -100, 2)
    for rc in (lib.vitm_distill(*rows, p, p, p, p, None, 0, 0, None), lib.vitm_distill_bwd(*rows, p, p, p, p, 0, 9, None)):
        assert rc == -1 and b"temperature" in lib.vitm_last_error()
