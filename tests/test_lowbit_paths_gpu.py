"""The 8-bit operators where the framework calls them: the VAE engine with AdamW, the generator with AdamW and 8-bit products,
and a training run of dense layers that uses all of them together."""
import numpy as np
import pytest
import torch

from oracle import lowbit_oracle as O
from test_engine_gpu import CASES, build_engine, load_fixed, make_case
from test_optim_gpu import f64, held

pytestmark = pytest.mark.gpu


def build(c, og, params, Wv, dtype, **kw):
    from conv1d_text_vae_amd import engine, geometry
    g = geometry.Geometry(c['T_in'], c['T_out'], og.input_vector_size, og.output_vector_size, c['n_filters'], c['k'], c['D'])
    return engine.VAEEngine(g, c['B'], Wv, dtype=dtype, device='cuda:0', weights=params, **kw)


@pytest.mark.parametrize('optimizer', ['adamw', 'adamw8'])
@pytest.mark.parametrize('use_graph', [False, True])
def test_engine_steps_follow_adamw(optimizer, use_graph):
    """Every step of the engine is AdamW on the gradients that it computed: clip at 10, lr 0.002, decay on kernels only.
    Tolerance as in test_optim_gpu.py."""
    c = CASES['mid']
    og, params, Wv, x, ids, eps, mask_e, mask_d = make_case(c, seed=1)
    eng = build(c, og, params, Wv, 'f32', optimizer=optimizer, weight_decay=0.1)
    load_fixed(eng, x, ids, eps, mask_e, mask_d)
    opt = eng.opt
    assert len(opt.params) == len(eng.seg_names)
    assert {w for n, w in zip(eng.seg_names, opt.weight_decay)} == {0.0, 0.1}
    eng.train_step(use_graph=use_graph, fixed_rng=True)           # (recording a step runs it once beside)
    for step in range(2, 5):
        before, p0 = held(opt), [f64(p) for p in opt.params]
        eng.train_step(use_graph=use_graph, fixed_rng=True)
        torch.cuda.synchronize()
        assert int(opt.t.item()) == step
        grads = [f64(eng.grads[eng.seg_off[n]:eng.seg_off[n] + p.numel()]) for n, p in zip(eng.seg_names, opt.params)]
        factor, norm = O.clip_factor(grads, 10.0)
        assert abs(float(eng.norm_out.item()) - norm) <= 2.0 ** -23 * norm
        for p, p_old, g, (m, v), wd, d in zip(opt.params, p0, grads, before, opt.weight_decay, opt._host):
            m, v = m[:d.n].astype(np.float64), v[:d.n].astype(np.float64)
            want, m1, v1 = O.adamw(p_old.reshape(-1), g, m, v, step, 0.002, 0.9, 0.999, 1e-7, wd, factor)
            # m' in fp32: three roundings of each term (they may cancel), the factor's fp32 rounding among them
            den = np.sqrt(v1 / (1 - 0.999 ** step)) + 1e-7
            tol = 4 * 2.0 ** -24 * np.abs(p_old.reshape(-1)) + 0.002 / (1 - 0.9 ** step) / den * (
                10 * 2.0 ** -23 * np.abs(m1) + 4 * 2.0 ** -24 * (0.9 * np.abs(m) + 0.1 * factor * np.abs(g)))
            assert (np.abs(f64(p).reshape(-1) - want) <= tol).all()
    eng.set_lr(0.5)
    assert eng.get_lr() == 0.5
    eng.reset_optimizer()
    assert int(opt.t.item()) == 0 and eng.get_lr() == 0.002 and not opt.moments(0)[1].any()


@pytest.mark.parametrize('optimizer', ['adamw', 'adamw8'])
def test_engine_forms_of_a_step_agree(optimizer, monkeypatch):
    """Eager, recorded list, HIP graph and the data-parallel sequence with one rank: the same weights and states, bit by bit."""
    c = CASES['mid']
    og, params, Wv, x, ids, eps, mask_e, mask_d = make_case(c, seed=2)
    got = []
    for form in ('eager', 'list', 'graph', 'buckets'):
        monkeypatch.setenv('C1V_STEP_LAUNCH', 'graph' if form == 'graph' else 'list')
        eng = build(c, og, params, Wv, 'bf16', optimizer=optimizer, force_bucketed=form == 'buckets', seed=5)
        load_fixed(eng, x, ids, eps, mask_e, mask_d)
        for _ in range(4):
            eng.train_step(use_graph=form != 'eager', fixed_rng=True, all_reduce=(lambda t: None) if form == 'buckets' else None)
        torch.cuda.synchronize()
        assert int(eng.step_ctr.item()) == 4 and int(eng.opt.t.item()) == 4
        got.append([eng.params.clone()] + [t.clone() for t in eng.opt.state_tensors()])
    for other in got[1:3]:
        for a, b in zip(got[0], other):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert (got[0][0] - got[3][0]).norm() <= 1e-3 * got[0][0].norm()          # (its weight gradients are summed in another order)


def test_warm_start_leaves_frozen_weights_alone():
    c = CASES['mid']
    og, params, Wv, x, ids, eps, mask_e, mask_d = make_case(c, seed=3)
    eng = build(c, og, params, Wv, 'bf16', optimizer='adamw8', weight_decay=0.5, frozen_encoder=True)
    load_fixed(eng, x, ids, eps, mask_e, mask_d)
    before = eng.get_weights()
    for _ in range(3):
        eng.train_step()
    after = eng.get_weights()
    for k in before:
        same = np.array_equal(before[k], after[k])
        assert same == k.startswith(('encoder_', 'z_')), k


def test_default_engine_keeps_nadam():
    c = CASES['tiny1']
    og, params, Wv, *_ = make_case(c)
    eng = build_engine(c, og, params, Wv, 'f32')
    assert eng.opt is None and eng.optimizer == 'nadam'
    with pytest.raises(ValueError):
        build(c, og, params, Wv, 'f32', optimizer='sgd')


# ---------------------------------------------------------------------------------------------------------------
# generator
# ---------------------------------------------------------------------------------------------------------------
def generator(products='fp8', optimizer='adamw8', units=96, **kw):
    from conv1d_text_vae_amd.seq2seq import Seq2SeqGenerator
    return Seq2SeqGenerator(text_size=9, feature_size=62, n_chars=23, units=units, lr=0.01, device='cuda:0', seed=1, optimizer=optimizer,
                            products=products, **kw)


def sentences(n=6, seed=0):
    rng = np.random.RandomState(seed)
    words = rng.standard_normal((n, 9, 62)).astype(np.float32)
    words[0, 4:] = 0.0
    words[1] = 0.0                                              # nothing survived: an empty text
    ids = rng.randint(0, 23, size=(n, 12))
    one = np.eye(23, dtype=np.float32)[ids]
    one[2, 5:] = 0.0
    return torch.from_numpy(words).cuda(), torch.from_numpy(one).cuda(), torch.from_numpy(np.roll(one, -1, axis=1).copy()).cuda()


class PlainLinear(torch.autograd.Function):
    """fp8.linear from its definition: torch products of the quantised values."""
    @staticmethod
    def forward(ctx, x, kernel, bias):
        ctx.save_for_backward(x, kernel)
        ctx.has_bias = bias is not None
        y = Q(x) @ Q(kernel.t()).t()
        return y if bias is None else y + bias

    @staticmethod
    def backward(ctx, dy):
        x, kernel = ctx.saved_tensors
        return Q(dy) @ Q(kernel).t(), Q(x.t()) @ Q(dy.t()).t(), dy.sum(0) if ctx.has_bias else None


def Q(x):
    return torch.from_numpy(O.quantized(f64(x)).astype(np.float32)).to(x.device)


def test_generator_gradients_with_8bit_products(monkeypatch):
    """The generator's loss and gradients against the same graph with the products from their definition.  Both sides work in
    fp32, 1e-6 or so apart; where that moves a value across a rounding border of e4m3 the value moves by up to 2^-3 of itself,
    which one value in 2^17 does: 1e-3 of the 2-norm covers hundreds of them."""
    from conv1d_text_vae_amd import fp8
    words, cin, cout = sentences()
    got = []
    for plain in (False, True):
        gen = generator(optimizer='rmsprop')
        if plain:
            monkeypatch.setattr(fp8, 'linear', lambda x, k, b=None: PlainLinear.apply(x.reshape(-1, x.shape[-1]), k, b).view(*x.shape[:-1], k.shape[1]))
        loss = gen.loss(words, cin, cout, train=True)           # same seed: the same dropout masks
        loss.backward()
        got.append((float(loss.detach()), {k: f64(v.grad) for k, v in gen.p.items()}))
    (la, ga), (lb, gb) = got
    assert abs(la - lb) < 1e-4 * abs(lb)
    for k in ga:
        assert np.linalg.norm(ga[k] - gb[k]) <= 1e-3 * np.linalg.norm(gb[k]), k
        assert np.abs(ga[k]).max() > 0


def test_generator_8bit_inference_follows_its_weights():
    """encode / decode_step with 8-bit products against the definition on the quantised weights, before and after an update."""
    words, cin, cout = sentences(seed=1)
    gen = generator()

    def check():
        with torch.no_grad():
            h = gen.encode(words)
            probs, h2 = gen.decode_step(cin[:, :3], h)
        x = f64(gen.attention(words))
        p = {k: f64(v) for k, v in gen.p.items()}

        def gru(name, x, h, masked):
            u = gen.U
            W, U, b = (p[name + s] for s in ('/kernel', '/recurrent_kernel', '/bias'))
            QW, QU = O.quantized(W.T).T, O.quantized(U.T).T
            xw = (O.quantized(x.reshape(-1, x.shape[-1])) @ QW).reshape(*x.shape[:2], 3 * u) + b
            hs = lambda a: np.clip(0.2 * a + 0.5, 0, 1)
            out = []
            for t in range(x.shape[1]):
                zr = O.quantized(h) @ QU[:, :2 * u]
                z, r = hs(xw[:, t, :u] + zr[:, :u]), hs(xw[:, t, u:2 * u] + zr[:, u:])
                new = z * h + (1 - z) * np.tanh(xw[:, t, 2 * u:] + O.quantized(r * h) @ QU[:, 2 * u:])
                live = (x[:, t] != 0).any(-1)[:, None] if masked else True
                h = np.where(live, new, h)
                out.append(h)
            return np.stack(out, 1), h
        want = gru('seq2seq_encoder_gru', x, np.zeros((x.shape[0], gen.U)), True)[1]
        # a state value that crosses a rounding border moves by 2^-4 of itself and goes on through the steps: bound in the 2-norm
        assert np.linalg.norm(f64(h) - want) <= 5e-3 * np.linalg.norm(want)
        assert not f64(h)[1].any()                              # the empty text keeps the zero state
        seq, want2 = gru('seq2seq_decoder_gru', f64(cin[:, :3]), f64(h), False)
        assert np.linalg.norm(f64(h2) - want2) <= 5e-3 * np.linalg.norm(want2)
        logits = O.quantized(seq.reshape(-1, gen.U)) @ O.quantized(p['seq2seq_decoder_dense/kernel'].T).T + p['seq2seq_decoder_dense/bias']
        e = np.exp(logits - logits.max(-1, keepdims=True))
        assert np.abs(f64(probs).reshape(-1, gen.C) - e / e.sum(-1, keepdims=True)).max() <= 2e-2
        return f64(h)
    a = check()
    for _ in range(3):
        gen.train_batch(words, cin, cout)                       # the weights move through raw pointers
    b = check()
    assert np.abs(a - b).max() > 1e-3
    gen.set_weights({'seq2seq_encoder_gru/bias': np.full(3 * gen.U, 0.1, dtype=np.float32)})
    check()
    assert gen.greedy_decode(torch.from_numpy(b.astype(np.float32)).cuda(), 0, 22, 7).shape[1] <= 8


def test_generator_8bit_weights_per_stream_update_and_graph():
    """The same answers from two streams and from a captured step, whoever quantised the weights first, and after updates by the
    optimizer alone (which the tensors' version counters tell)."""
    words, cin, cout = sentences(seed=2)
    gen, warm = generator(), generator()
    h0 = torch.zeros(cin.shape[0], gen.U, device='cuda')
    with torch.no_grad():
        want = warm.decode_step(cin[:, :2], h0)                 # the same seed, the same weights
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):                           # the first call of this generator: nothing of the graph is kept
            out = gen.decode_step(cin[:, :2], h0)
        eager = gen.decode_step(cin[:, :2], h0)
        assert all(torch.equal(a, b) for a, b in zip(eager, want))
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = gen.decode_step(cin[:, :2], h0)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(other, want))
    versions = [v._version for v in gen.p.values()]
    gen.opt.step([torch.ones_like(v) for v in gen.p.values()])
    assert all(v._version > n for v, n in zip(gen.p.values(), versions))
    with torch.no_grad():
        moved = gen.decode_step(cin[:, :2], h0)
        warm.set_weights(gen.get_weights())
        again = warm.decode_step(cin[:, :2], h0)
        assert not torch.equal(moved[1], want[1]) and all(torch.equal(a, b) for a, b in zip(moved, again))
        graph.replay()                                          # computes with the weights of its time
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, again))


def test_generator_training_loss_without_gradients_is_the_same():
    """The training form (dropout, whole-sequence products in 8 bits) under no_grad: the loss of the same seed, to the bit."""
    words, cin, cout = sentences(seed=4)
    with_graph = generator().loss(words, cin, cout, train=True)
    with torch.no_grad():
        assert torch.equal(generator().loss(words, cin, cout, train=True), with_graph.detach())


def test_generator_8bit_inference_sees_every_change_of_its_weights():
    """Updates that the tensors' version counters do not tell -- a replayed optimizer step, a write through `.data`, a replaced
    `.data` -- between decoded characters: each time the answers of a fresh generator with the same weights."""
    words, cin, cout = sentences(seed=3)
    gen, fresh = generator(), generator()
    h0 = torch.zeros(cin.shape[0], gen.U, device='cuda')

    def check():
        fresh.set_weights(gen.get_weights())
        with torch.no_grad():
            got, want = gen.decode_step(cin[:, :2], h0), fresh.decode_step(cin[:, :2], h0)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            assert torch.equal(gen.encode(words), fresh.encode(words))
            assert np.array_equal(gen.greedy_decode(got[1], 0, 22, 5), fresh.greedy_decode(want[1], 0, 22, 5))
        assert torch.equal(gen.eval_batch(words, cin, cout), fresh.eval_batch(words, cin, cout))
        return got[1]
    grads = [torch.ones_like(v) for v in gen.p.values()]
    seen = [check()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gen.opt.step(grads)
    seen.append(check())
    assert torch.equal(seen[0], seen[1])                        # (capturing is no step)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        seen.append(check())
    gen.p['seq2seq_decoder_gru/kernel'].data.mul_(-1.5)
    seen.append(check())
    gen.p['seq2seq_decoder_gru/recurrent_kernel'].data = gen.p['seq2seq_decoder_gru/recurrent_kernel'].detach() * 0.5
    seen.append(check())
    assert all(not torch.equal(a, b) for a, b in zip(seen[1:], seen[2:]))


@pytest.mark.parametrize('products', ['f32', 'fp8'])
@pytest.mark.parametrize('optimizer', ['adamw', 'adamw8'])
def test_generator_trains_with_adamw(products, optimizer):
    words, cin, cout = sentences(seed=2)
    gen = generator(products, optimizer, weight_decay=0.0)
    start = gen.get_weights()
    for i in range(4):
        if i == 2:
            gen.lr = 0.02                                       # as ReduceLROnPlateau does
        loss = gen.train_batch(words, cin, cout)
        assert torch.isfinite(loss)
    assert int(gen.opt.t.item()) == 4 and gen.opt.get_lr() == 0.02
    assert all((gen.get_weights()[k] != start[k]).any() for k in start)
    assert np.isfinite(float(gen.eval_batch(words, cin, cout)))
    assert all(gen.opt.weight_decay[i] == 0.0 for i in range(len(gen.p)))


def test_estimator_with_8bit_training_and_serving(fasttext_small):
    from conv1d_text_vae_amd import Conv1dTextVAE
    X, y, emb = fasttext_small
    np.random.seed(3)
    vae = Conv1dTextVAE(emb, emb, max_epochs=2, batch_size=2, n_filters=16, latent_dim=8)
    vae.vae_optimizer, vae.generator_optimizer, vae.generator_products = 'adamw8', 'adamw8', 'fp8'
    vae.fit(X, y)
    assert vae._generator.products == 'fp8' and vae._vae_runtime.optimizer == 'adamw8'
    assert np.isfinite(vae.vae_history_[-1]['val_loss']) and np.isfinite(vae.seq2seq_history_[-1]['val_loss'])
    out = vae.predict(X[:2])
    assert len(out) == 2 and all(isinstance(s, str) and s for s in out)
    assert 'vae_optimizer' not in vae.get_params()


@pytest.fixture(scope='module')
def fasttext_small():
    from conv1d_text_vae_amd import Conv1dTextVAE, DefaultTokenizer
    from conv1d_text_vae_amd import embeddings as E
    from test_estimator_cpu import load_testdata
    X, y = load_testdata(max_target_words=10)
    tok = DefaultTokenizer()
    words = [w for t in list(X) + list(y) for w in Conv1dTextVAE.tokenize(t, tok.tokenize_into_words(t))]
    return X, y, E.synthetic_fasttext(words, vector_size=20, bucket=500, seed=7)


# ---------------------------------------------------------------------------------------------------------------
# all of them together
# ---------------------------------------------------------------------------------------------------------------
def test_a_run_of_all_of_them():
    """Two dense layers trained for some steps (linear forward and backward, AdamW with 8-bit states), then served (weights
    quantised once, one row and many): every step's gradients against the definition, the parameters through the optimizer's
    own check, the served outputs against the layers."""
    from conv1d_text_vae_amd import fp8, optim
    from test_optim_gpu import check_step
    gen = torch.Generator('cuda').manual_seed(4)
    rnd = lambda *s: torch.randn(*s, generator=gen, device='cuda')
    k1, b1, k2, b2 = 0.1 * rnd(150, 260), 0.1 * rnd(260), 0.1 * rnd(260, 33), 0.1 * rnd(33)
    leaves = [t.requires_grad_(True) for t in (k1, b1, k2, b2)]
    wd = [0.01, 0.0, 0.01, 0.0]
    opt = optim.AdamW(leaves, lr=0.01, weight_decay=wd, clipnorm=1.0, states='8bit', seed=8)
    for step in range(4):
        x, target = rnd(77, 150), rnd(77, 33)
        h = torch.relu(fp8.linear(x, k1, b1))
        y = fp8.linear(h, k2, b2)
        d = (y - target) / 77
        grads = torch.autograd.grad(y, leaves, d)
        X, H, D = f64(x), f64(h), f64(d)
        dh = (O.quantized(D) @ O.quantized(f64(k2)).T) * (H > 0)
        want = [O.quantized(X.T) @ O.quantized(dh.T).T, dh.sum(0), O.quantized(H.T) @ O.quantized(D.T).T, D.sum(0)]
        for g, w in zip(grads, want):
            assert np.linalg.norm(f64(g) - w) <= 1e-3 * np.linalg.norm(w)      # (rounding borders of dh, as above)
        check_step(opt, list(grads), 0.01, wd, 1.0)
    with torch.no_grad():
        q1, q2 = fp8.quantize_cols(k1), fp8.quantize_cols(k2)
        x = rnd(40, 150)
        many = fp8.dense(fp8.dense(x, q1, b1, relu=True), q2, b2)
        train = fp8.linear(torch.relu(fp8.linear(x, k1, b1)), k2, b2)
        assert (many - train).norm() <= 1e-3 * train.norm()
        for i in (0, 39):
            one = fp8.dense(fp8.dense(x[i:i + 1], q1, b1, relu=True), q2, b2)
            assert (one - many[i:i + 1]).norm() <= 1e-2 * many[i].norm()       # (a border crossed in one row weighs more)
