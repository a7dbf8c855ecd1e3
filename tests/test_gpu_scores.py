"""Class-score operators on a real MI355X against their definitions in 64 bits (score_oracle.py).

Tolerances count roundings.  u = 2^-24 is half a step of fp32; a sum of V positive terms passes at most 64 additions in a
thread, 6 in a wave, 15 across waves and one a segment; an exponential of t is off by 3 u |t| (difference, scale, product) and
its own unit; the final rounding to the logits' type is half a step, finfo.eps / 2."""
import pytest
import torch

import score_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
BF, F32 = torch.bfloat16, torch.float32
NINF = float("-inf")


@pytest.fixture(scope="module")
def log_probs():
    from vitm_amd import log_probs
    return log_probs


@pytest.fixture(scope="module")
def Loss():
    from vitm_amd.training import DistillationLoss
    return DistillationLoss


def _gen(seed):
    return torch.Generator(device="cpu").manual_seed(seed)


def _scores(R, V, dtype, seed, scale=3.0):
    return (torch.randn(R, V, generator=_gen(seed)) * scale).to(DEV).to(dtype)


def _spread(z, T):
    """max |z - max| / T of each row over its finite scores, at most 200 (beyond that an exponential is 0), and |max| / T."""
    z = z.double()
    fin = z.isfinite()
    m = torch.where(fin, z, torch.full_like(z, -1e300)).amax(1)
    m = torch.where(fin.any(1), m, torch.zeros_like(m))
    low = torch.where(fin, z, m[:, None].expand_as(z)).amin(1)
    return ((m - low) / T).clamp(max=200), m.abs() / T


def _near(got, ref, tol, what):
    """Equal where the reference is not finite, else within tol.  A reference beyond fp32's range, 2^128 (1 - 2^-24) =
    3.4028e38, is an infinity in the fp32 output: fp32's lowest value over a temperature of 0.5 is -6.8e38."""
    got, ref = got.double(), ref.double()
    ref = torch.where(ref.abs() > torch.finfo(F32).max, torch.sign(ref) * float("inf"), ref)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    odd = ~ref.isfinite()
    assert torch.equal(got[odd].nan_to_num(7e300, 8e300, 9e300), ref[odd].nan_to_num(7e300, 8e300, 9e300)), what
    err, tol = (got - ref).abs()[~odd], tol.expand_as(ref)[~odd]
    if err.numel():
        assert got[~odd].isfinite().all(), what
        worst = (err / tol).max().item()
        assert worst <= 1, f"{what}: {worst:.2f} times the tolerance"


def _check_log_probs(z, targets, r, top_k, T):
    z2 = z.reshape(-1, z.shape[-1])
    t2 = None if targets is None else targets.reshape(z2.shape[0], -1).long()
    o = O.log_probs(z2, t2, top_k, T)
    rng, m = _spread(z2, T)
    tol = U * (160 + 4 * rng)
    if targets is not None:
        _near(r.logprobs.reshape(t2.shape), o["logprobs"], tol[:, None], "logprobs")
    _near(r.lse.reshape(-1), o["lse"], tol + 2 * U * m, "lse")
    if r.entropy is not None:
        _near(r.entropy.reshape(-1), o["entropy"], tol * (1 + o["entropy"]), "entropy")
    if top_k:
        assert torch.equal(r.top_indices.reshape(-1, top_k), o["top_indices"])
        _near(r.top_logprobs.reshape(-1, top_k), o["top_logprobs"], tol[:, None], "top_logprobs")
    return o, rng


SHAPES = [(1, 1), (1000, 3), (65, 33), (130, 60), (37, 120), (9, 129), (3, 2), (5, 7), (33, 10), (300, 1000), (4, 511), (4, 513), (2, 2048), (2, 2049), (3, 4097), (7, 5000),
          (600, 5003), (3, 16384), (3, 16391), (2, 40001), (1, 131072), (513, 20001), (2, 70001),
          (1, 300007), (515, 66001), (2, 500000)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("R,V", SHAPES)
def test_log_probs_and_gradient(log_probs, R, V, dtype):
    T = (1.0, 0.7, 2.0)[(R + V) % 3]
    K = min(V, (0, 1, 5, 20, 64, 128)[(3 * R + V) % 6])
    G = 1 + (R + V) % 3
    z = _scores(R, V, dtype, R * 1000 + V).requires_grad_(True)
    tgt = torch.randint(0, V, (R, G), generator=_gen(V)).to(DEV)
    if R > 2:
        tgt[1, 0] = -100
        tgt[2, -1] = tgt[2, 0]
    r = log_probs(z, tgt, top_k=K, entropy=True, temperature=T)
    o, rng = _check_log_probs(z.detach(), tgt, r, K, T)
    g = [torch.randn(t.shape, generator=_gen(5)).to(DEV) for t in (r.logprobs, r.lse, r.entropy)]
    heads = [r.logprobs, r.lse, r.entropy]
    if K:
        g.append(torch.randn(R, K, generator=_gen(6)).to(DEV))
        heads.append(r.top_logprobs)
    (dz,) = torch.autograd.grad(heads, z, g)
    ref, mag = O.log_probs_grad(o, tgt, T, g[0], g[1], g[2], g[3] if K else None)
    assert dz.dtype == dtype
    n = G + K
    _near(dz, ref, U * (200 + n + 6 * rng[:, None]) * mag + torch.finfo(dtype).eps / 2 * ref.abs() * 1.01 + 1e-37, "dlogits")


@pytest.mark.parametrize("which", ["logprobs", "lse", "entropy", "top"])
def test_log_probs_gradient_of_each_output_alone(log_probs, which):
    R, V, K = 6, 3001, 9
    z = _scores(R, V, F32, 4).requires_grad_(True)
    tgt = torch.randint(0, V, (R, 1), generator=_gen(1)).to(DEV)
    r = log_probs(z, tgt, top_k=K, entropy=True)
    head = dict(logprobs=r.logprobs, lse=r.lse, entropy=r.entropy, top=r.top_logprobs)[which]
    up = torch.randn(head.shape, generator=_gen(2)).to(DEV)
    (dz,) = torch.autograd.grad(head, z, up)
    o = O.log_probs(z.detach(), tgt, K, 1.0)
    kw = {dict(logprobs="g_lp", lse="g_lse", entropy="g_ent", top="g_top")[which]: up}
    ref, mag = O.log_probs_grad(o, tgt, 1.0, **kw)
    rng, _ = _spread(z.detach(), 1.0)
    _near(dz, ref, U * (220 + 6 * rng[:, None]) * mag + U * ref.abs() + 1e-37, which)


def test_log_probs_gradient_against_differences(log_probs):
    """fp32, a step of 2^-6: the quotient of the float64 values at the two ends, which the operator's gradient must match up to
    the third derivative (|f'''| <= 8 for a sum of log probabilities and an entropy below 3 nats)."""
    z0 = _scores(1, 9, F32, 8, scale=1.0)
    tgt = torch.tensor([[4]], device=DEV)
    z = z0.clone().requires_grad_(True)
    r = log_probs(z, tgt, entropy=True)
    (dz,) = torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), z)
    h = 2.0 ** -6
    f = lambda z: (lambda o: (o["logprobs"].sum() + o["entropy"].sum()).item())(O.log_probs(z, tgt, 0, 1.0))
    for i in range(9):
        e = torch.zeros_like(z0, dtype=torch.float64)
        e[0, i] = h
        d = (f(z0.double() + e) - f(z0.double() - e)) / (2 * h)
        assert abs(dz[0, i].item() - d) <= 8 * h * h / 6 + 1e-5


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [1, 3, 10, 16, 25, 31, 33, 58, 64, 65, 121, 128, 129, 250])
def test_short_rows(log_probs, V, dtype):
    """Several rows a wave, up to the sizes where the next form takes over, with rows that start anywhere in a granule; the number
    of rows does not fill the last workgroup."""
    for R, off, pad in ((1, 0, 0), (70, 0, 0), (67, 3, 5), (1025, 1, 0)):
        z = _scores(R, V + off + pad, dtype, V + R)[:, off:off + V]
        tgt = torch.randint(0, V, (R, 2), generator=_gen(V)).to(DEV)
        for ent in (True, False):
            _check_log_probs(z, tgt, log_probs(z, tgt, entropy=ent, temperature=0.7), 0, 0.7)


VIEWS = {
    "padded rows": lambda b: b(7, 1016)[:, :1003],
    "offset": lambda b: b(7, 1016)[:, 5:1008],
    "token slice": lambda b: b(4, 6, 523)[:, :-1],
    "both strides": lambda b: b(4, 6, 640)[:, 1:, 3:523],
    "every other row": lambda b: b(8, 2501)[::2],
    "one row": lambda b: b(2600)[1:],
    "transposed": lambda b: b(301, 9).t(),
    "every other class": lambda b: b(6, 602)[:, ::2],
    "expanded": lambda b: b(1, 777).expand(5, 777),
    "swapped": lambda b: b(5, 4, 333).transpose(0, 1),
    "four dimensions": lambda b: b(2, 3, 4, 77)[:, :2, :3],
    "long odd rows": lambda b: b(3, 33001)[:, 1:],
}


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("view", sorted(VIEWS))
def test_views(log_probs, Loss, view, dtype):
    """Strided, offset and misaligned rows: the same bits as of a contiguous copy whose rows start alike, gradients included."""
    base = lambda *s: (torch.randn(*s, generator=_gen(11)) * 2).to(DEV).to(dtype)
    z = VIEWS[view](base)
    lead, V = z.shape[:-1], z.shape[-1]
    R = z.numel() // V
    tgt = torch.randint(0, V, lead, generator=_gen(3)).to(DEV)
    zr = z.detach().requires_grad_(True)
    r = log_probs(zr, tgt, top_k=7, entropy=True)
    assert r.logprobs.shape == r.lse.shape == r.entropy.shape == lead and r.top_indices.shape == (*lead, 7)
    o, rng = _check_log_probs(z, tgt, r, 7, 1.0)
    up = torch.randn(lead, generator=_gen(4)).to(DEV)
    (dz,) = torch.autograd.grad(r.logprobs, zr, up)
    ref, mag = O.log_probs_grad(o, tgt.reshape(R, 1), 1.0, g_lp=up.reshape(R, 1))
    half = torch.finfo(dtype).eps / 2 * 1.01
    _near(dz.reshape(R, V), ref, U * (220 + 6 * rng[:, None]) * mag + half * ref.abs() + 1e-37, "dlogits")
    K = 5
    idx = torch.stack([torch.randperm(V, generator=_gen(i))[:K] for i in range(R)]).to(DEV)
    tl = torch.log_softmax(torch.randn(R, K + 1, generator=_gen(9)), 1)[:, :K].to(DEV)
    loss, dz = Loss(temperature=2.0, label_weight=0.3, tail=True, reduction="none").loss_and_grad(
        z, tl.view(*lead, K), idx.view(*lead, K), tgt)
    _check_distill(z.reshape(R, V), tl, idx, tgt.reshape(R), loss.reshape(R), dz.reshape(R, V), 2.0, 0.3, True)


# ---- masks, infinities, ties --------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [40, 3000, 40000])
def test_masked_rows(log_probs, V, dtype):
    low = torch.finfo(dtype).min
    z = _scores(8, V, dtype, V)
    z[0] = NINF                                   # nothing left
    z[1, 1:] = NINF                               # one class left
    z[2] = low                                    # the lowest finite value everywhere: uniform
    z[3, V // 2:] = low                           # masked with the lowest value
    z[4, torch.randperm(V, generator=_gen(1))[:V - 12]] = NINF
    z[5, :V - 3] = NINF
    z[6] = 0.0
    z[6, ::2] = -0.0                              # both zeros are equal
    K = 20
    tgt = torch.zeros(8, 2, dtype=torch.int64, device=DEV)
    tgt[:, 1] = V - 1
    for T in (1.0, 0.5):
        zr = z.clone().requires_grad_(True)
        r = log_probs(zr, tgt, top_k=K, entropy=True, temperature=T)
        o, rng = _check_log_probs(z, tgt, r, K, T)
        g = torch.randn(8, generator=_gen(2)).to(DEV)
        (dz,) = torch.autograd.grad([r.entropy, r.lse], zr, [g, g])
        ref, mag = O.log_probs_grad(o, tgt, T, g_ent=g, g_lse=g)
        _near(dz, ref, U * (220 + 6 * rng[:, None]) * mag + torch.finfo(dtype).eps / 2 * 1.01 * ref.abs() + 1e-37, "dlogits")
        assert (dz[0] == 0).all()


@pytest.mark.parametrize("V", [40, 3000, 40000])
def test_nan_and_inf_rows(log_probs, Loss, V):
    z = _scores(4, V, F32, V)
    z[1, V // 3] = float("nan")
    z[2, V // 2] = float("inf")
    tgt = torch.full((4,), V - 1, device=DEV)
    zr = z.clone().requires_grad_(True)
    r = log_probs(zr, tgt, top_k=5, entropy=True)
    for t in (r.logprobs, r.entropy, r.lse, r.top_logprobs):
        assert t[1].isnan().all() and t[2].isnan().all() and t[0].isfinite().all() and t[3].isfinite().all()
    assert (r.top_indices[1:3] == -1).all() and (r.top_indices[[0, 3]] >= 0).all()
    (dz,) = torch.autograd.grad(r.logprobs.sum(), zr)
    assert dz[1].isnan().any() and dz[0].isfinite().all() and dz[3].isfinite().all()
    idx = torch.arange(6, device=DEV).expand(4, 6)
    tl = torch.log_softmax(torch.zeros(4, 6, device=DEV), 1)
    loss, dz = Loss(reduction="none").loss_and_grad(z, tl, idx)
    assert loss[1:3].isnan().all() and loss[[0, 3]].isfinite().all() and dz[[0, 3]].isfinite().all()


def _ordered(kind, V):
    i = torch.arange(V, dtype=torch.float32)
    if kind == "equal":
        return torch.full((V,), 1.25)
    if kind == "rising":
        return i / 64
    if kind == "falling":
        return -i / 64
    if kind == "two values":
        return (torch.rand(V, generator=_gen(1)) < 0.5).float()
    if kind == "few large":
        return torch.where(torch.rand(V, generator=_gen(2)) < 0.003, 3.0, -2.0)
    if kind == "one thread":                      # the best classes a stride apart, so that one thread holds them
        z = torch.randn(V, generator=_gen(3))
        z[5::2048] += 50
        z[6::2048] += 50
        return z
    if kind == "half equal best":
        return torch.where(torch.rand(V, generator=_gen(4)) < 0.5, torch.full((V,), 2.0), torch.randn(V, generator=_gen(5)))
    if kind == "all but one masked":
        z = torch.full((V,), NINF)
        z[V - 1] = 0.0
        return z
    raise KeyError(kind)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [100, 1999, 16000, 50000])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "two values", "few large", "one thread", "half equal best",
                                  "all but one masked"])
def test_top_order(log_probs, kind, V, dtype):
    """Orders and ties that defeat a bound taken from groups of threads: still the K largest, the lower class first."""
    z = _ordered(kind, V).to(DEV).to(dtype).expand(3, V).contiguous()
    z[1] = z[1].roll(17)
    z[2] = z[2].flip(0)
    for K in (1, 33, 100):
        _check_log_probs(z, None, log_probs(z, top_k=K), K, 1.0)


def test_targets_outside_the_classes(log_probs):
    z = _scores(5, 50, F32, 1).requires_grad_(True)
    tgt = torch.tensor([3, 50, -1, -100, 2 ** 40], device=DEV)
    r = log_probs(z, tgt)
    assert r.logprobs.isnan().tolist() == [False, True, True, False, True] and r.logprobs[3] == 0
    (dz,) = torch.autograd.grad(r.logprobs, z, torch.ones(5, device=DEV))
    assert dz.isfinite().all() and (dz[1:] == 0).all() and (dz[0] != 0).any()
    assert log_probs(z.detach(), tgt.clamp(0, 49).int()).logprobs.isfinite().all()


def test_ignore_index_that_is_a_class(log_probs, Loss):
    """A padding class as the ignored one: its rows count as ignored, everywhere."""
    z = _scores(4, 30, F32, 1).requires_grad_(True)
    tgt = torch.tensor([[5, 0], [0, 0], [7, 7], [0, 3]], device=DEV)
    r = log_probs(z, tgt, ignore_index=0)
    assert (r.logprobs[tgt == 0] == 0).all() and (r.logprobs[tgt != 0] != 0).all()
    (dz,) = torch.autograd.grad(r.logprobs.sum(), z)
    assert (dz[1] == 0).all() and (dz[0] != 0).any()
    tl, idx = _teacher(4, 30, 3, 1)
    loss, dz = Loss(label_weight=0.5, reduction="none", ignore_index=0).loss_and_grad(z.detach(), tl, idx, tgt[:, 1].contiguous())
    assert loss[0] == 0 and loss[1] == 0 and (dz[:2] == 0).all() and (loss[2:] != 0).all()


def test_empty_and_shapes(log_probs, Loss):
    z = torch.zeros(0, 7, device=DEV, requires_grad=True)
    r = log_probs(z, torch.zeros(0, 2, dtype=torch.int64, device=DEV), top_k=3, entropy=True)
    assert torch.autograd.grad(r.logprobs.sum() + r.entropy.sum() + r.top_logprobs.sum(), z)[0].shape == (0, 7)
    z = torch.zeros(3, 7, device=DEV, requires_grad=True)
    r = log_probs(z, torch.zeros(3, 0, dtype=torch.int64, device=DEV))
    assert r.logprobs.shape == (3, 0)
    assert (torch.autograd.grad(r.logprobs.sum() + r.lse.sum(), z)[0] > 0).all()
    r = log_probs(torch.zeros(0, 7, device=DEV), torch.zeros(0, dtype=torch.int64, device=DEV), top_k=3, entropy=True)
    assert r.logprobs.shape == (0,) and r.top_indices.shape == (0, 3) and r.entropy.shape == (0,)
    r = log_probs(torch.zeros(7, device=DEV), torch.tensor(2, device=DEV), top_k=2)
    assert r.logprobs.shape == () and r.top_indices.tolist() == [0, 1] and r.entropy is None
    r = log_probs(torch.zeros(2, 3, 7, device=DEV), torch.zeros(2, 3, 4, dtype=torch.int64, device=DEV))
    assert r.logprobs.shape == (2, 3, 4) and r.lse.shape == (2, 3) and r.top_indices is None
    z = torch.zeros(0, 7, device=DEV, requires_grad=True)
    e = (torch.zeros(0, 2, device=DEV), torch.zeros(0, 2, dtype=torch.int64, device=DEV))
    loss = Loss()(z, *e)
    assert loss.item() == 0 and torch.autograd.grad(loss, z)[0].shape == (0, 7)
    loss, dz = Loss().loss_and_grad(z, *e)
    assert loss.item() == 0 and dz.shape == (0, 7)


def test_offsets_beyond_32_bits(log_probs, Loss):
    """Rows more than 2^31 elements apart."""
    step = 2 ** 31 + 8
    store = torch.empty(step + 4096, dtype=BF, device=DEV)
    z = store.as_strided((2, 3001), (step, 1), 0)
    z.copy_(_scores(2, 3001, BF, 3))
    tgt = torch.tensor([7, 3000], device=DEV)
    r = log_probs(z, tgt, top_k=6, entropy=True)
    _check_log_probs(z, tgt, r, 6, 1.0)
    idx = torch.tensor([[1, 5, 2900], [0, 2, 3000]], device=DEV)
    tl = torch.log_softmax(torch.randn(2, 4, generator=_gen(1)), 1)[:, :3].to(DEV)
    loss, dz = Loss(tail=True, reduction="none").loss_and_grad(z, tl, idx, tgt)
    _check_distill(z, tl, idx, tgt, loss, dz, 1.0, 0.0, True)


# ---- distillation -------------------------------------------------------------------------------------------------
def _check_distill(z, tl, idx, labels, loss, dz, T, a, tail, up=None):
    """Row losses and the gradient of sum up_r loss_r."""
    ref, mag, rdz, gm = O.distill(z, tl, idx, labels, T, a, tail)
    rng, _ = _spread(z, T)
    rng1, _ = _spread(z, 1.0)
    c = 320 + 8 * torch.maximum(rng, rng1 if a > 0 else rng)
    if loss is not None:
        _near(loss, ref, U * c * mag + 1e-37, "loss")
    if dz is not None:
        if up is not None:
            rdz, gm = rdz * up.double()[:, None], gm * up.double().abs()[:, None]
        half = torch.finfo(dz.dtype).eps / 2 * 1.01
        _near(dz, rdz, U * c[:, None] * gm + half * rdz.abs() + 1e-37, "dlogits")
    return ref, mag, c


def _teacher(R, V, K, seed, ragged=True, rest=True):
    idx = torch.stack([torch.randperm(V, generator=_gen(seed + i))[:K] for i in range(R)])
    t = torch.randn(R, K + 1, generator=_gen(seed)) * 2
    tl = torch.log_softmax(t, 1)[:, :K] if rest else torch.log_softmax(t[:, :K], 1)
    if ragged and K > 1:
        idx[::3, -1] = -1
    return tl.to(DEV), idx.to(DEV)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("R,V", SHAPES)
def test_distillation(Loss, R, V, tail, dtype):
    """Every reduction, eager gradient and fused gradient, over all the row sizes."""
    T = (1.0, 2.0, 0.8)[(R + V) % 3]
    a = (0.0, 0.3, 1.0, 0.5)[(R * 7 + V) % 4]
    K = max(1, min(V // 2, (1, 5, 20, 64, 128)[(R + 2 * V) % 5]))
    z = _scores(R, V, dtype, R + V, scale=2.0)
    tl, idx = _teacher(R, V, K, V)
    labels = torch.randint(0, V, (R,), generator=_gen(V + 1)).to(DEV)
    labels[::5] = -100
    if R > 3:
        labels[3] = idx[3, 0]                     # a label inside the list
    n = max(1, int((labels != -100).sum()))
    loss, dz = Loss(T, a, tail, "none").loss_and_grad(z, tl, idx, labels)
    ref, mag, c = _check_distill(z, tl, idx, labels, loss, dz, T, a, tail)
    tot = U * ((c + R) * mag).sum() + U * R * ref.abs().sum() + 1e-37
    for red, div in (("sum", 1), ("mean", n)):
        up = torch.full((R,), 1.0 / div, device=DEV)
        loss, dz = Loss(T, a, tail, red).loss_and_grad(z, tl, idx, labels)
        _near(loss, ref.sum() / div, tot / div, red)
        _check_distill(z, tl, idx, labels, None, dz, T, a, tail, up)
        zr = z.clone().requires_grad_(True)
        l2 = Loss(T, a, tail, red)(zr, tl, idx, labels)
        _near(l2.detach(), ref.sum() / div, tot / div, red)      # its sums may be taken in another order
        (d2,) = torch.autograd.grad(l2 * -1.5, zr)
        _check_distill(z, tl, idx, labels, None, d2, T, a, tail, up * -1.5)
        assert torch.equal(Loss(T, a, tail, red)(z, tl, idx, labels), l2.detach())
    zr = z.clone().requires_grad_(True)
    up = torch.randn(R, generator=_gen(3)).to(DEV)
    l3 = Loss(T, a, tail, "none")(zr, tl, idx, labels)
    _check_distill(z, tl, idx, labels, l3.detach(), None, T, a, tail)
    (d3,) = torch.autograd.grad(l3, zr, up)
    _check_distill(z, tl, idx, labels, None, d3, T, a, tail, up)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("V", [12, 2500, 30000])
def test_distillation_odd_lists(Loss, V, tail):
    """Listed twice, absent entries, entries of probability 0, nothing listed, everything listed, mass near 1, indices and labels
    outside the classes, masked students."""
    R, K = 12, 6
    z = _scores(R, V, F32, V)
    tl, idx = _teacher(R, V, K, 5, ragged=False)
    labels = torch.randint(0, V, (R,), generator=_gen(2)).to(DEV)
    idx[0, 1] = idx[0, 4] = idx[0, 0]             # the same class three times
    idx[1, :] = -1                                # nothing listed
    tl[2, 3] = NINF                               # an entry of probability 0
    tl[3, :] = NINF
    tl[4] = torch.log_softmax(tl[4].double(), 0).float()   # the list holds all of the teacher's mass
    labels[5] = -100
    labels[6] = V                                 # refused rows
    idx[7, 2] = V
    idx[8, 2] = -2
    z[9] = NINF                                   # a student with no class left
    z[10, :] = NINF                               # a student with classes only inside the list
    z[10, idx[10]] = torch.randn(K, generator=_gen(4)).to(DEV)
    labels[10] = idx[10, 2]
    labels[11] = idx[11, 5]
    for T, a in ((1.0, 0.0), (2.0, 0.4), (1.0, 1.0)):
        loss, dz = Loss(T, a, tail, "none").loss_and_grad(z, tl, idx, labels)
        _check_distill(z, tl, idx, labels, loss, dz, T, a, tail)
        assert (dz[5:10] == 0).all() and loss[5] == 0 and loss[9] == 0 and loss[6:9].isnan().all()
        zr = z.clone().requires_grad_(True)
        l2 = Loss(T, a, tail, "none")(zr, tl, idx, labels)
        (d2,) = torch.autograd.grad(l2, zr, torch.ones(R, device=DEV))
        _check_distill(z, tl, idx, labels, l2.detach(), d2, T, a, tail)
    if V == 12:                                   # every class listed: no tail
        idx = torch.stack([torch.randperm(V, generator=_gen(i)) for i in range(R)]).to(DEV)
        tl = torch.log_softmax(torch.randn(R, V, generator=_gen(7)), 1).to(DEV)
        z = _scores(R, V, F32, 8)
        loss, dz = Loss(1.0, 0.0, tail, "none").loss_and_grad(z, tl, idx)
        _check_distill(z, tl, idx, None, loss, dz, 1.0, 0.0, tail)


def test_distillation_tail_of_tiny_mass(Loss):
    """The student's mass outside the list far below fp32's unit: the tail's loss and gradient keep their digits."""
    V, K = 5000, 4
    z = _scores(3, V, F32, 2, scale=1.0)
    tl, idx = _teacher(3, V, K, 9, ragged=False)
    z.scatter_(1, idx, 60.0)
    loss, dz = Loss(1.0, 0.0, True, "none").loss_and_grad(z, tl, idx)
    _check_distill(z, tl, idx, None, loss, dz, 1.0, 0.0, True)
    assert (loss > 1).all()


def test_distillation_of_itself_is_zero(log_probs, Loss):
    """A student equal to its teacher, with the tail: loss 0 and gradient 0 up to rounding."""
    z = _scores(9, 7001, F32, 1)
    for T in (1.0, 3.0):
        top = log_probs(z, top_k=50, temperature=T)
        loss, dz = Loss(T, 0.0, True, "none").loss_and_grad(z, top.top_logprobs, top.top_indices)
        _check_distill(z, top.top_logprobs, top.top_indices, None, loss, dz, T, 0.0, True)
        assert loss.abs().max() <= T * T * U * 2000 and dz.abs().max() <= T * U * 2000


def test_all_rows_ignored(Loss):
    z = _scores(6, 100, BF, 1)
    tl, idx = _teacher(6, 100, 5, 1)
    loss, dz = Loss(label_weight=0.5).loss_and_grad(z, tl, idx, torch.full((6,), -100, device=DEV))
    assert loss.item() == 0 and (dz == 0).all()


def test_teacher_in_bf16_and_int32_indices(Loss):
    z = _scores(6, 100, BF, 1)
    tl, idx = _teacher(6, 100, 5, 1)
    a = Loss()(z, tl.to(BF), idx.int())
    assert torch.equal(a, Loss()(z, tl.to(BF).float(), idx))


# ---- memory, streams, graphs, repeatability -----------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V,off,ldd", [(13, 0, 13), (100, 3, 129), (2501, 1, 2503), (20001, 5, 20016)])
def test_gradients_stay_in_their_rows(V, off, ldd, dtype):
    """Gradients written with a pitch and an alignment of their own: right, and nothing outside the rows is touched."""
    from vitm_amd import _lib, _score_ops as S
    lib = _lib.load()
    R, K = 5, 3
    z = _scores(R, V, dtype, V)
    rows = S.rows_of(z)
    tl, idx = _teacher(R, V, K, 3)
    st = torch.cuda.current_stream().cuda_stream
    stats = torch.empty(R, 2, device=DEV)
    lse, g = torch.empty(R, device=DEV), torch.randn(R, generator=_gen(1)).to(DEV)
    _lib.check(lib.vitm_log_probs(*rows.args(), 1.0, None, 0, -100, 0, None, lse.data_ptr(), None, None, None, stats.data_ptr(),
                                  st), "lp")
    row_loss, state = torch.empty(R, device=DEV), torch.empty(R * 8, device=DEV)
    for what in ("log_probs", "distill"):
        buf = torch.full((off + R * ldd + 64,), 99.0, device=DEV).to(dtype)
        out = buf.as_strided((R, V), (ldd, 1), off)
        if what == "log_probs":
            _lib.check(lib.vitm_log_probs_bwd(*rows.args(), 1.0, None, 0, -100, None, 0, stats.data_ptr(), None, None, g.data_ptr(),
                                              None, None, out.data_ptr(), 0, ldd, st), "bwd")
            o = O.log_probs(z, None, 0, 1.0)
            ref, mag = O.log_probs_grad(o, None, 1.0, g_lse=g)
            rng, _ = _spread(z, 1.0)
            _near(out, ref, U * (220 + 6 * rng[:, None]) * mag + torch.finfo(dtype).eps / 2 * 1.01 * ref.abs() + 1e-37, what)
        else:
            _lib.check(lib.vitm_distill(*rows.args(), 1.0, 0.0, 1, tl.data_ptr(), idx.data_ptr(), K, None, -100, 0, row_loss.data_ptr(),
                                        None, None, state.data_ptr(), out.data_ptr(), 0, ldd, st), "distill")
            _check_distill(z, tl, idx, None, row_loss, out, 1.0, 0.0, True)
        left = torch.ones_like(buf, dtype=torch.bool)
        left.as_strided((R, V), (ldd, 1), off).fill_(False)
        assert (buf[left] == 99).all(), what


def _calls(log_probs, Loss, z, tl, idx, tgt):
    def fn():
        r = log_probs(z, tgt, top_k=8, entropy=True)
        loss, dz = Loss(2.0, 0.3, True).loss_and_grad(z, tl, idx, tgt)
        l2, d2 = Loss(1.0, 0.0, False, "sum").loss_and_grad(z, tl, idx)
        return [*r, loss, dz, l2, d2]
    return fn


@pytest.mark.parametrize("R,V,dtype", [(6, 50, F32), (700, 1000, BF), (5, 70001, BF), (300, 24001, F32)])
def test_repeatable_and_captured(log_probs, Loss, R, V, dtype):
    """Equal calls give equal bits, on another stream and from a graph replayed between eager work too; a graph follows its
    inputs."""
    z = _scores(R, V, dtype, 2)
    tl, idx = _teacher(R, V, 9, 2)
    tgt = torch.randint(0, V, (R,), generator=_gen(2)).to(DEV)
    fn = _calls(log_probs, Loss, z, tl, idx, tgt)
    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))
    first = fn()
    assert same(first, fn())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)             # the call must wait for its own stream's work, not the default stream's
        z2 = z.clone()
        other = _calls(log_probs, Loss, z2, tl, idx, tgt)()
    torch.cuda.current_stream().wait_stream(side)
    assert same(first, other)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):                            # two graphs of the same calls
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(fn())
        graphs.append(graph)
    for step in range(3):
        z.copy_(_scores(R, V, dtype, 20 + step))
        for gr in graphs:
            gr.replay()
        eager = fn()
        torch.cuda.synchronize()
        for out in outs:
            assert same(out, eager), step


def test_second_derivative_is_refused(log_probs, Loss):
    """Also where the upstream gradient is a constant: a penalty on the gradient would otherwise be left out in silence."""
    z = _scores(4, 10, F32, 1).to(DEV).requires_grad_(True)
    y = torch.zeros(4, dtype=torch.int64, device=DEV)
    tl, ti = torch.log_softmax(z.detach(), -1).topk(3)
    for f in (lambda: log_probs(z, y).logprobs.sum(), lambda: Loss()(z, tl, ti)):
        plain, = torch.autograd.grad(f(), z)
        (dz,) = torch.autograd.grad(f(), z, create_graph=True)
        assert torch.equal(dz, plain)
        with pytest.raises(RuntimeError, match="no second derivative"):
            (z.sum() + dz.pow(2).sum()).backward()


def test_backward_twice_from_one_graph(log_probs, Loss):
    """retain_graph: the second backward sees what the first saw; an input changed in place in between is refused."""
    z = _scores(4, 3000, F32, 1).requires_grad_(True)
    tl, idx = _teacher(4, 3000, 6, 1)
    loss = Loss(tail=True)(z, tl, idx) + log_probs(z, entropy=True).entropy.sum()
    (a,) = torch.autograd.grad(loss, z, retain_graph=True)
    (b,) = torch.autograd.grad(loss, z, retain_graph=True)
    assert torch.equal(a, b)
    with torch.no_grad():
        z.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(loss, z)


# ---- together, in the framework's own paths -----------------------------------------------------------------------
def _model(seed, depth=2, classes=10):
    import torch.nn as nn
    from vitm_amd.models import VITC, VisionTransformer
    torch.manual_seed(seed)
    LN = nn.LayerNorm
    return VITC(VisionTransformer(32, patch_size=8, num_classes=classes, num_heads=2, mlp_ratio=2.0, depth=depth, embed_dim=64,
                                  norm_layer=LN, final_norm_layer=LN)).to(DEV)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_classify(dtype):
    m = _model(1, classes=37).to(dtype)
    x = torch.randn(9, 3, 32, 32, generator=_gen(1)).to(DEV).to(dtype)
    y = torch.randint(0, 37, (9,), generator=_gen(2)).to(DEV)
    with torch.no_grad():
        logits = m(x)
    r = m.classify(x, labels=y, entropy=True)
    _check_log_probs(logits, y, r, 5, 1.0)
    assert m.classify(x, top_k=100).top_indices.shape == (9, 37)
    assert m.classify(x[:0], labels=y[:0]).top_indices.shape == (0, 5)


@pytest.mark.parametrize("tail", [False, True])
def test_training_step_with_a_teacher(log_probs, tail):
    """Teacher's forward -> its best classes -> loss and gradient -> backward: the step's gradients are those of the same loss
    through autograd's graph of the logits, and a stored teacher gives the same step."""
    from vitm_amd import training
    x = torch.randn(8, 3, 32, 32, generator=_gen(1)).to(DEV)
    y = torch.randint(0, 10, (8,), generator=_gen(2)).to(DEV)
    y[3] = -100
    teacher = _model(7, depth=1)
    fn = training.DistillationLoss(temperature=2.0, label_weight=0.3, tail=tail)
    with torch.no_grad():
        top = log_probs(teacher(x), top_k=4, temperature=2.0)
    ref = _model(3)
    loss = fn(ref(x), top.top_logprobs, top.top_indices, y)
    loss.backward()

    def step(**kw):
        m = _model(3)
        tr = training.Trainer(m, training.AdamW(m.parameters(), lr=1e-3), distillation=fn, max_norm=1e9,
                              **({} if "teacher_top" in kw else dict(teacher=teacher, teacher_top_k=4)))
        return m, tr, tr.step(x, y, **kw)

    m, tr, l1 = step()
    assert abs(l1.item() - loss.item()) <= 1e-5 * abs(loss.item())   # two orders of the same sums: about 400 u of it each
    for p, q in zip(m.parameters(), ref.parameters()):
        assert (p.grad - q.grad).abs().max() <= 1e-5 * q.grad.abs().max() + 1e-12
    m2, _, l2 = step(teacher_top=(top.top_logprobs, top.top_indices))
    assert torch.equal(l1, l2) and all(torch.equal(a, b) for a, b in zip(m.parameters(), m2.parameters()))
    with pytest.raises(ValueError, match="teacher returned"):
        training.Trainer(m2, training.AdamW(m2.parameters()), distillation=fn, teacher=_model(1, classes=12)).step(x, y)
    with pytest.raises(RuntimeError, match="teacher or teacher_top"):
        training.Trainer(m2, training.AdamW(m2.parameters()), distillation=fn).step(x, y)
    with pytest.raises(ValueError, match="teacher_top needs"):
        training.Trainer(m2, training.AdamW(m2.parameters())).step(x, y, teacher_top=(top.top_logprobs, top.top_indices))


@pytest.mark.parametrize("stored", [False, True])
def test_graphed_training_step_with_a_teacher(log_probs, stored):
    """The captured step: bit for bit the eager one, several replays."""
    from vitm_amd import training, GraphedTrainStep
    teacher = _model(7, depth=1)
    fn = training.DistillationLoss(temperature=2.0, label_weight=0.3, tail=True)
    batches = [(torch.randn(8, 3, 32, 32, generator=_gen(i)).to(DEV), torch.randint(0, 10, (8,), generator=_gen(50 + i)).to(DEV))
               for i in range(6)]

    def run(graphed):
        m = _model(3)
        tr = training.Trainer(m, training.AdamW(m.parameters(), lr=1e-3), distillation=fn, teacher=None if stored else teacher,
                              teacher_top_k=4)
        g = GraphedTrainStep(tr) if graphed else tr
        losses = []
        for x, y in batches:
            kw = {}
            if stored:
                with torch.no_grad():
                    top = log_probs(teacher(x), top_k=4, temperature=2.0)
                kw["teacher_top"] = (top.top_logprobs, top.top_indices)
            losses.append(g.step(x, y, **kw).clone())
        return losses, list(m.parameters()), g, kw

    (l1, p1, _, _), (l2, p2, g, kw) = run(False), run(True)
    assert all(torch.equal(a, b) for a, b in zip(l1, l2)) and all(torch.equal(a, b) for a, b in zip(p1, p2))
    with pytest.raises(RuntimeError, match="captured with"):
        x, y = batches[0]
        g.step(x, y) if stored else g.step(x, y, teacher_top=(torch.zeros(8, 4, device=DEV), torch.zeros(8, 4, dtype=torch.int64,
                                                                                                        device=DEV)))


def test_graphed_step_refuses_a_teacher_that_changed():
    from vitm_amd import training, GraphedTrainStep
    teacher, m = _model(7, depth=1), _model(3, depth=1)
    tr = training.Trainer(m, training.AdamW(m.parameters(), lr=1e-3), distillation=training.DistillationLoss(), teacher=teacher)
    g = GraphedTrainStep(tr, warmup=1)
    x, y = torch.randn(8, 3, 32, 32, generator=_gen(1)).to(DEV), torch.randint(0, 10, (8,), generator=_gen(2)).to(DEV)
    for _ in range(3):
        g.step(x, y)
    before = [p.detach().clone() for p in m.parameters()]
    with torch.no_grad():
        next(teacher.parameters()).mul_(0.5)
    with pytest.raises(RuntimeError, match="teacher's weights"):
        g.step(x, y)
    assert all(torch.equal(a, b) for a, b in zip(before, m.parameters()))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_gradient_interleaved_with_the_logits(dtype):
    """Rows of logits and gradient in turn, in one buffer: their spans meet, the rows do not."""
    from vitm_amd import _lib
    lib = _lib.load()
    R, V, K = 5, 1001, 3
    buf = torch.zeros(R, 2 * V, device=DEV, dtype=dtype)
    z, out = buf[:, :V], buf[:, V:]
    z.copy_(_scores(R, V, dtype, 3))
    kept = z.clone()
    tl, idx = _teacher(R, V, K, 3)
    row_loss = torch.empty(R, device=DEV)
    _lib.check(lib.vitm_distill(z.data_ptr(), _lib.BF16 if dtype == BF else _lib.F32, 0, 2 * V, R, R, V, 1.0, 0.0, 1, tl.data_ptr(),
                                idx.data_ptr(), K, None, -100, 0, row_loss.data_ptr(), None, None, None, out.data_ptr(), 0, 2 * V,
                                torch.cuda.current_stream().cuda_stream), "distill")
    assert torch.equal(z, kept)
    _check_distill(z, tl, idx, None, row_loss, out, 1.0, 0.0, True)


def test_very_many_short_rows(log_probs, Loss):
    """More rows than 1024 threads each would leave room for."""
    R, V = (1 << 22) + 3, 10
    z = torch.randn(R, V, generator=torch.Generator(DEV).manual_seed(1), device=DEV)
    idx = torch.arange(3, device=DEV).expand(R, 3)
    tl = torch.log_softmax(z[:, :4] * 0.5, 1)[:, :3].contiguous()
    labels = torch.arange(R, device=DEV) % V
    labels[::7] = -100
    loss, dz = Loss(2.0, 0.5, True, "none").loss_and_grad(z, tl, idx, labels)
    for a in (0, R // 2, R - 1000):               # (the oracle takes 64 bits a class)
        part = slice(a, a + 1000)
        _check_distill(z[part], tl[part], idx[part], labels[part], loss[part], dz[part], 2.0, 0.5, True)
    n = int((labels != -100).sum())
    mean, dm = Loss(2.0, 0.5, True).loss_and_grad(z, tl, idx, labels)
    # a thread adds 4097 rows, then 6 + 15 across the workgroup; each row's loss counts as it is
    _near(mean, loss.double().sum() / n, U * 4200 * loss.double().abs().sum() / n, "mean")
    assert (dm - dz / n).abs().max() <= 4 * U * dz.abs().max() / n


@pytest.mark.parametrize("R", [2, 777, 1024, 1025, 4100])
def test_the_mean_is_that_of_the_rows(Loss, R):
    """The sum of the rows' losses is taken in 64 bits and divided once: off the losses' mean by its own rounding, half a step."""
    z = _scores(R, 40, F32, R)
    tl, idx = _teacher(R, 40, 6, 1)
    for labels in (None, torch.where(torch.arange(R, device=DEV) % 5 == 1, -100, 3)):
        for red, n in (("sum", 1), ("mean", R if labels is None else int((labels != -100).sum()))):
            rows = Loss(2.0, 0.0, False, "none")(z, tl, idx, labels).double()
            exact = rows.sum() / n
            got = Loss(2.0, 0.0, False, red)(z, tl, idx, labels)
            assert (got.double() - exact).abs() <= exact.abs() * U * 1.0001, (red, labels is None)


@pytest.mark.parametrize("T", [4.0, 8.0, 9.0, 30.0, 1000.0, 10000.0])
@pytest.mark.parametrize("R,V,K,tail,kind", [(64, 100, 100, False, ""), (64, 100, 100, True, ""), (64, 100, 20, True, ""), (64, 100, 99, False, ""),
                                             (16, 5000, 64, True, ""), (16, 5000, 100, False, "masked"), (3, 40001, 100, True, ""),
                                             (5, 40001, 128, False, "masked"), (16, 900, 30, True, "twice")])
def test_distillation_at_high_temperatures(log_probs, Loss, R, V, K, tail, kind, T):
    """The divergence shrinks with T^2 while its terms do not: the loss keeps its digits all the same.

    With the listed classes apart (the tail form, or T above 8) all of the divergence's terms q d - q + p are positive and good to
    some 30 u each.  The sums over the row are off by eps = 180 u at most (see above), which moves mass between list and rest:
    eps |p_rest - q_rest| and eps^2 in the divergence; q_rest = 1 - sum q, of 7 + 1 additions and q good to 2 u, counts with
    its d: 12 u |d_rest|.  Otherwise ln s is off by eps, and so is the divergence.  (A class listed twice has no small d.)"""
    z, zt = _scores(R, V, F32, V, scale=2.0), _scores(R, V, F32, V + 1, scale=2.0)
    if kind == "masked":                          # what the list leaves out is masked: its mass is 0 and has to come out so
        z[:, K:] = NINF
        zt[:, K:] = NINF
    top = log_probs(zt, top_k=K, temperature=T)
    tl, idx = top.top_logprobs, top.top_indices.clone()
    if kind == "twice":
        idx[:, 1] = idx[:, 0]
    ref, mag, _, _ = O.distill(z, tl, idx, None, T, 0.0, tail)
    p = torch.softmax(z.double() / T, 1)
    listed = torch.zeros_like(p).scatter_(1, idx, 1.0) > 0
    p_rest = torch.where(listed, torch.zeros_like(p), p).sum(1)
    q_rest = (1 - tl.double().exp().sum(1)).clamp(min=0) if tail else torch.zeros_like(p_rest)
    d = torch.where((q_rest > 0) & (p_rest > 0), (q_rest.log() - p_rest.log()).abs(), torch.zeros_like(p_rest))
    eps = 180 * U
    kl_tol = 30 * U * ref.abs() / T ** 2 + eps ** 2
    if tail:
        kl_tol = kl_tol + eps * (p_rest - q_rest).abs() + 12 * U * d
    elif T > 8:
        kl_tol = kl_tol + eps * p_rest
    else:
        kl_tol = kl_tol + eps
    if kind == "twice":
        kl_tol = kl_tol + 40 * U
    loss, dz = Loss(T, 0.0, tail, "none").loss_and_grad(z, tl, idx)
    _near(loss, ref, T ** 2 * kl_tol, "loss")
    _check_distill(z, tl, idx, None, None, dz, T, 0.0, tail)
    zr = z.clone().requires_grad_(True)
    l2 = Loss(T, 0.0, tail, "none")(zr, tl, idx)
    _near(l2.detach(), ref, T ** 2 * kl_tol, "loss")
    (d2,) = torch.autograd.grad(l2, zr, torch.ones(R, device=DEV))
    _check_distill(z, tl, idx, None, None, d2, T, 0.0, tail)


@pytest.mark.parametrize("R", [1023, 1024, 1025, 2049, 4100])
@pytest.mark.parametrize("V,tail", [(7, False), (300, True)])
def test_distillation_of_many_rows(Loss, R, V, tail):
    """On both sides of 1024 rows: up to there every workgroup counts the labels itself, beyond a kernel counts them first, in
    rounds of 1024, and the total adds several rows a thread.  Ignored labels lie in every round, so that a round left out or
    counted twice shows."""
    T, a, K = 2.0, 0.4, 3
    z = _scores(R, V, F32, R)
    idx = torch.stack([torch.randperm(V, generator=_gen(i % 64))[:K] for i in range(R)]).to(DEV)
    tl = torch.log_softmax(torch.randn(R, K + 1, generator=_gen(R)), 1)[:, :K].to(DEV)
    labels = torch.randint(0, V, (R,), generator=_gen(1))
    labels[torch.rand(R, generator=_gen(2)) < torch.arange(R) / R] = -100      # few at first, most at the end
    labels = labels.to(DEV)
    n = int((labels != -100).sum())
    each = Loss(T, a, tail, "none")(z, tl, idx, labels)
    ref, mag, c = _check_distill(z, tl, idx, labels, each, None, T, a, tail)
    for red, div in (("mean", n), ("sum", 1)):
        up = torch.full((R,), 1.0 / div, device=DEV)
        want = each.double().sum() / div
        loss, dz = Loss(T, a, tail, red).loss_and_grad(z, tl, idx, labels)
        _near(loss, want, 2 * U * (c * mag).sum() / div + U * want.abs(), red)   # its rows' sums may be taken in another order
        _check_distill(z, tl, idx, labels, None, dz, T, a, tail, up)
        zr = z.clone().requires_grad_(True)
        l2 = Loss(T, a, tail, red)(zr, tl, idx, labels)
        assert torch.equal(l2.detach(), Loss(T, a, tail, red)(z, tl, idx, labels))
        (d2,) = torch.autograd.grad(l2, zr)
        _check_distill(z, tl, idx, labels, None, d2, T, a, tail, up)
    loss, dz = Loss(T, a, tail).loss_and_grad(z, tl, idx, torch.full_like(labels, -100))
    assert loss == 0 and (dz == 0).all()


@pytest.mark.parametrize("R,V,dtype", [(1500, 300, BF), (2100, 33, F32)])
def test_many_rows_captured(log_probs, Loss, R, V, dtype):
    """The count of the rows in memory, from a graph replayed several times between eager work."""
    z = _scores(R, V, dtype, 2)
    idx = torch.stack([torch.randperm(V, generator=_gen(i % 50))[:9] for i in range(R)]).to(DEV)
    tl = torch.log_softmax(torch.randn(R, 10, generator=_gen(9)), 1)[:, :9].to(DEV)
    tgt = torch.randint(0, V, (R,), generator=_gen(2)).to(DEV)
    fn = _calls(log_probs, Loss, z, tl, idx, tgt)
    first = fn()
    assert all(torch.equal(a, b) for a, b in zip(first, fn()))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    for step in range(4):
        z.copy_(_scores(R, V, dtype, 20 + step))
        tgt[step::7] = -100                       # another count each time
        graph.replay()
        eager = fn()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), step


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("top_k", [0, 1])
@pytest.mark.parametrize("z0", [0.0, -3.0])
def test_logarithms_of_exact_sums(log_probs, dtype, top_k, z0):
    """V equal classes: every exponential is 1 and their sum V exactly, so that lse = z0 + ln V, log p = -ln V and the entropy
    ln V are off by the logarithm (its hardware form good to 2^-24 in [0.5, 1), times ln 2 that is off by 2^-25 of it: 2^-24 in all)
    and the final rounding alone."""
    for V in [2, 3, 5, 7, 10, 11, 13, 37, 100, 101, 997, 1000, 1001, 3001, 4093, 10007, 21001, 50021, 99991, 131071, 300007]:
        r = log_probs(torch.full((2, V), z0, device=DEV, dtype=dtype), torch.zeros(2, dtype=torch.int64, device=DEV), top_k=top_k,
                      entropy=True)
        ln = torch.log(torch.tensor(float(V), dtype=torch.float64, device=DEV))
        for got, want in ((r.lse, z0 + ln), (r.logprobs, -ln), (r.entropy, ln), (r.top_logprobs, -ln)):
            if got is not None:
                assert ((got.double() - want).abs() <= U * want.abs() + U).all(), (V, got, want)
