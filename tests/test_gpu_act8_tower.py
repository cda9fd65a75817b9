"""The per-layer tower with its activations kept in 8 bits (act_dtype=fp8): every gradient of a step against
the formula in 64 bits on the tower's own operands, the kept codes against the default tower's activations,
runs of steps as graphs against eager ones."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(synth, layers, keep, B, act_dtype, params, **kw):
    from hipfm.models.deepfm import NativeDeepFM
    m = NativeDeepFM(synth.feature_size, synth.F, 8, layers, keep, batch_size=B, device=DEV, init=False, fused=False,
                     learning_rate=1e-3, act_dtype=act_dtype, **kw)
    m.load_tf_params(params)
    return m


def setup(layers, B, steps=1, seed=3):
    from hipfm.data.synthetic import make_synth
    from hipfm.models.reference import init_params
    synth = make_synth("total:20000", seed=seed)
    params = init_params(synth.feature_size, synth.F, 8, layers, False, seed=seed)
    return synth, params, [synth.batch(B, step=s, device=DEV, id_dtype=torch.int32) for s in range(steps)]


def dsum(a, b):
    """a^T b and the bound of its fp32 accumulation in any order, in 64 bits."""
    a, b = a.double().cpu(), b.double().cpu()
    return a.t() @ b, (a.shape[0] + 2) * 2.0 ** -24 * (a.abs().t() @ b.abs())


@pytest.mark.parametrize("layers,keep,B", [([96, 64], [0.5, 0.5], 100), ([64, 160], [1.0, 0.8], 300),
                                           ([1024, 256], [0.9, 1.0], 640), ([256, 1024], [0.5, 1.0], 513)])
def test_step_gradients_match_the_formula(layers, keep, B):
    from hipfm.ops import act8 as A8
    synth, params, data = setup(layers, B)
    m, d = (make(synth, layers, keep, B, t, params) for t in ("fp8", "bf16"))
    wt = m.WT16[1].clone()                                 # (the optimizer refreshes it)
    m.train_step(*data[0])
    d.train_step(*data[0])
    torch.cuda.synchronize()
    m.check_errors()
    # the forward pass is the default tower's; its kept activations are the codes of the same values
    want = A8.pack(d.H[0])
    assert torch.equal(m.H8[0].codes, want.codes) and torch.equal(m.H8[0].scales, want.scales)
    assert torch.equal(m.H[1], d.H[1]) and torch.equal(m.dZ[1], d.dZ[1]) and torch.equal(m.prob, d.prob)
    x8 = A8.unpack(m.H8[0], torch.float32)
    assert torch.equal(x8 > 0, d.H[0] > 0)
    g = {n: m.g[s.off:s.off + int(torch.Size(s.shape).numel())].view(s.shape).double().cpu()
         for n, s in m.dense_segs.items()}
    for i, x in ((1, x8), (0, m.E)):
        w, bound = dsum(m.dZ[i], x)
        assert ((g[f"Deep-part/mlp{i}/weights"] - w).abs() <= bound).all()
        b, bound = dsum(m.dZ[i], torch.ones(m.M, 1))
        assert ((g[f"Deep-part/mlp{i}/biases"] - b[:, 0]).abs() <= bound[:, 0]).all()
    N = m.Np[0]
    prod, bound = dsum(m.dZ[1].t(), wt.view(N, m.Np[1]).t())
    s = 1.0 / keep[0]
    prod, bound = s * prod, s * bound
    bound = bound + 2.0 ** -23 * prod.abs()                 # (the scale's own rounding and its product's)
    dz = torch.where(x8.double().cpu() > 0, prod, torch.zeros(()).double())
    assert ((m.dZ[0].double().cpu() - dz).abs() <= bound + 2.0 ** -8 * (prod.abs() + bound)).all()
    assert (m.dZ[0].cpu()[dz == 0] == 0).all() and (dz != 0).any()


@pytest.mark.parametrize("opt,layers", [("Adam", [1024, 512, 1024]), ("ftrl", [96, 64])])
def test_graph_steps_equal_eager_steps(opt, layers):
    B, keep = 512, [0.5] * len(layers)
    synth, params, data = setup(layers, B, steps=3)
    a, b = (make(synth, layers, keep, B, "fp8", params, optimizer=opt, sparse_update="lazy") for _ in range(2))
    for r in range(3):                                     # (the second and third rounds replay)
        for x in data:
            a.train_step(*x)
            b.train_step(*x, use_graph=True)
        torch.cuda.synchronize()
        assert torch.equal(a.p, b.p), r
        assert torch.equal(a.tv[:synth.feature_size], b.tv[:synth.feature_size]), r
    b.check_errors()
    assert torch.isfinite(a.p).all()


def test_a_larger_batch_and_evaluation():
    """Buffers grow with the batch; evaluation between steps leaves the next step's result as it is."""
    layers, keep = [96, 64, 96], [0.5, 0.5, 0.5]
    synth, params, data = setup(layers, 400, steps=2)
    a, b = (make(synth, layers, keep, 128, "fp8", params) for _ in range(2))
    for m in (a, b):
        m.train_step(*(t[:100].contiguous() for t in data[0]))
    p = a.predict(*data[1][:2])
    assert p.shape[0] == 400
    for m in (a, b):
        m.train_step(*data[1])
    torch.cuda.synchronize()
    assert torch.equal(a.p, b.p) and a.H8[0].codes.shape[0] == 512


def test_no_transposed_copies():
    """Neither kept nor written: the gradient products take rows."""
    layers, B = [1024, 256], 300
    synth, params, data = setup(layers, B)
    m = make(synth, layers, [1.0, 1.0], B, "fp8", params)
    m.train_step(*data[0])
    torch.cuda.synchronize()
    m.check_errors()
    assert m.Et is None and m.Ht is None and m.dZt is None


@pytest.mark.parametrize("layers,keep", [([96, 160, 64], [0.5, 1.0, 0.8]), ([1024, 256, 512], [0.9, 0.5, 1.0]),
                                         ([64, 160, 96, 32], [1.0, 0.5, 0.5, 1.0]), ([256, 1024, 128, 512], [0.5, 0.9, 1.0, 0.5])])
def test_layers_that_share_buffers(layers, keep):
    """H and dZ of layers two apart lie in one buffer, at other widths.  Every layer's dZ, as its weight gradient takes it,
    against the product of the layer above's in 64 bits, and its gradients against those of this dZ and the default tower's
    activations; in a second step too, whose batch leaves rows of the first one's behind it."""
    from hipfm.ops import act8 as A8
    synth, params, (first, second) = setup(layers, 601, steps=2)
    m, d = (make(synth, layers, keep, 601, t, params) for t in ("fp8", "bf16"))
    taken, wgrad = {}, m._wgrad_act8

    def keep_dz(i):
        taken[i] = m.dZ[i].clone()
        wgrad(i)

    m._wgrad_act8 = keep_dz
    for batch in (first, [t[:333].contiguous() for t in second]):
        wts = [w.clone() for w in m.WT16]                      # (the optimizer refreshes them)
        for t in (m, d):
            t.train_step(*batch)
        torch.cuda.synchronize()
        m.check_errors()
        g = {n: m.g[s.off:s.off + int(torch.Size(s.shape).numel())].view(s.shape).double().cpu()
             for n, s in m.dense_segs.items()}
        assert torch.equal(m.prob, d.prob) and torch.equal(m.E, d.E)
        top = len(layers) - 1
        assert torch.equal(taken[top], d.dZ[top])
        for i in reversed(range(top + 1)):
            x = A8.unpack(A8.pack(d.H[i - 1]), torch.float32) if i else m.E
            for what, right in (("weights", x), ("biases", torch.ones(m.M, 1, device=DEV))):
                w, bound = dsum(taken[i], right)
                got = g[f"Deep-part/mlp{i}/{what}"]
                assert ((got - w.view(got.shape)).abs() <= bound.view(got.shape)).all(), (i, what)
            if i:
                s = 1.0 / keep[i - 1]
                prod, bound = dsum(taken[i].t(), wts[i].view(m.Np[i - 1], m.Np[i]).t())
                prod, bound = s * prod, s * bound + 2.0 ** -23 * s * prod.abs()      # (the scale's own rounding and its product's)
                on = x.double().cpu() > 0
                want = torch.where(on, prod, torch.zeros(()).double())
                assert ((taken[i - 1].double().cpu() - want).abs() <= bound + 2.0 ** -8 * (prod.abs() + bound)).all(), i
                assert (taken[i - 1].cpu()[~on] == 0).all() and on.any(), i
        # the second step starts from the same parameters
        d.p.copy_(m.p)
        d.rec.copy_(m.rec)
        d.refresh_shadows()
