"""Sampling decode of the engine: encoder, decoder steps, vocabulary projection (bf16 or 8 bits) and drawing together.  Every step's words are
checked against the definition in 64 bits on the logits that the step left in the workspace, those of the 8-bit projection against the
quantised operands."""
import numpy as np
import pytest
import torch

from test_gpu_parity import SPECS, build
from test_gpu_serving import lp_bound, product_bound, quant_oracle, sample_oracle

pytestmark = pytest.mark.gpu
EOS, PAD = 1, 0
# vocabularies of the larger one-launch rows, and beyond them: the steps then share the workspace's scratch
LONG = dict(channels={401: 6}, decimation=3, enc_embed=5, enc_rnn=[4, 6], dec_embed=3, dec_rnn=12, vocab=9001, aux_layer=None, ff_dropout=0.0,
            rnn_dropout=0.0)
LONGEST = dict(LONG, vocab=20001)


def network(name, B=19, L=6, seed=5):
    eng, ws, ospec, P, batch = build(dict(SPECS, long=LONG, longest=LONGEST)[name], B, 26, L, seed=seed)
    return eng, ws


def uniforms(L, B, seed=0):
    return torch.rand(L, B, generator=torch.Generator(device='cuda').manual_seed(seed), device='cuda')


def check_steps(eng, ws, hyp, score, u, steps, **kw):
    B, L, V = ws['B'], ws['L'], eng.spec.vocab
    hyp, score, u = hyp.cpu().numpy(), score.double().cpu().numpy(), u.double().cpu().numpy()
    logits = ws['proj']['out'].view(L, B, V).double().cpu().numpy()
    col = {n: np.broadcast_to(v.double().cpu().numpy() if isinstance(v, torch.Tensor) else float(np.float32(v)), (B,))
           for n, v in dict(dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **kw).items()}
    fed = ws['U'].view(L, B).cpu().numpy()
    assert (fed[0] == EOS).all() and (hyp[:, steps:] == PAD).all()
    for b in range(B):
        done, total, bound = False, 0.0, 0.0
        for l in range(steps):
            tok, lp = sample_oracle(logits[l, b], u[l, b], col['temperature'][b], col['top_k'][b], col['top_p'][b], col['min_p'][b])
            assert hyp[b, l] == (PAD if done else tok)
            assert l + 1 >= L or fed[l + 1, b] == tok
            if not done:
                total += lp
                bound += lp_bound(lp, V) + abs(total) * 2.0 ** -24          # (the sum rounds once a step)
            done = done or tok == EOS
        assert abs(score[b] - total) <= bound * (1 + 2.0 ** -20)


@pytest.mark.parametrize('int8', [False, True])
@pytest.mark.parametrize('name', ['tiny_odd', 'small_dropout', 'cat_aux_hidden_proj', 'long', 'longest'])
def test_every_step_draws_by_the_definition(name, int8):
    eng, ws = network(name)
    B, L = ws['B'], ws['L']
    g = torch.Generator(device='cuda').manual_seed(3)
    mixed = dict(temperature=torch.rand(B, generator=g, device='cuda') * 2, top_k=torch.randint(0, 12, (B,), generator=g, device='cuda'),
                 top_p=torch.rand(B, generator=g, device='cuda') + 0.3, min_p=torch.rand(B, generator=g, device='cuda') * 0.4 - 0.2)
    for i, kw in enumerate([dict(), dict(temperature=0.6, top_k=7, top_p=0.9, min_p=0.05), mixed]):
        u = uniforms(L, B, i)
        hyp, score = eng.sample_decode(ws, u, which='p', int8_projection=int8, **kw)
        check_steps(eng, ws, hyp, score, u, L, **kw)
    u = uniforms(4, B, 9)
    hyp, score = eng.sample_decode(ws, u, which='p', int8_projection=int8, max_len=4, temperature=3.0)
    check_steps(eng, ws, hyp, score, u, 4, temperature=3.0)


@pytest.mark.parametrize('name,B', [('tiny_odd', 19), ('small_dropout', 1), ('small_dropout', 19), ('cat_aux_hidden_proj', 19), ('cfg2_widths', 130)])
def test_int8_projection(name, B):
    """Its logits are the product of the quantised state rows and weights, the biases added in fp32."""
    eng, ws = network(name, B=B)
    L, V, pr = ws['L'], eng.spec.vocab, eng.proj
    eng.sample_decode(ws, uniforms(L, B), which='p', int8_projection=True)
    fin = pr.sizes[-2]
    qw, sw = quant_oracle(pr.WT[-1][:, :fin].double().cpu().numpy())
    bias = eng.store.view('proj%d.b' % (pr.nl - 1))
    for l in range(L):
        if pr.nl == 1:
            h = ws['dec']['Yext'].view(-1, eng.dec.ldy)[(l + 1) * B:(l + 2) * B, :fin]
        else:
            h = ws['proj']['act'][-1][l * B:(l + 1) * B, :fin]
        q, s = quant_oracle(h.double().cpu().numpy())
        acc = (q.astype(np.int64) @ qw.astype(np.int64).T).astype(np.float64)
        want = acc * s.astype(np.float64)[:, None] * sw.astype(np.float64)[None] + bias.double().cpu().numpy().reshape(-1)[None]
        got = ws['proj']['out'].view(L, B, V)[l].double().cpu().numpy()
        assert (np.abs(got - want) <= product_bound(acc, s.astype(np.float64), sw.astype(np.float64), bias, want, torch.float32)).all()


@pytest.mark.parametrize('name', ['tiny_odd', 'cat_aux_hidden_proj'])
def test_temperature_zero_is_greedy(name):
    eng, ws = network(name)
    want = eng.greedy_decode(ws, which='p').clone()
    hyp, score = eng.sample_decode(ws, uniforms(ws['L'], ws['B']), temperature=0.0, which='p')
    assert torch.equal(hyp, want) and not score.any()
    # and with 8-bit weights the greedy words are those of a beam of one
    hyp = eng.sample_decode(ws, uniforms(ws['L'], ws['B']), temperature=0.0, which='p', int8_projection=True)[0].clone()
    beam, _ = eng.beam_decode(ws, 1, which='p', int8_projection=True)
    assert torch.equal(hyp, beam)


@pytest.mark.parametrize('int8', [False, True])
@pytest.mark.parametrize('name', ['small_dropout', 'cat_aux_hidden_proj', 'long', 'longest'])
def test_one_graph_serves_all_numbers_settings_and_weights(name, int8):
    eng, ws = network(name)
    L, B = ws['L'], ws['B']
    for i, kw in enumerate([dict(), dict(top_k=3), dict(temperature=1.5, top_p=0.7), dict(min_p=0.2)]):
        u = uniforms(L, B, i)
        if i == 2:
            ws['X'].mul_(-0.5)
        if i == 3:
            for _ in range(3):
                eng.train_step(ws)                       # other weights: the 8-bit image and the token table are made anew
            eng.pack('p')
        hyp, score = eng.sample_decode(ws, u, which='p', int8_projection=int8, **kw)
        hyp, score = hyp.clone(), score.clone()
        check_steps(eng, ws, hyp, score, u, L, **kw)
        for _ in range(2):
            h, s = eng.sample_decode(ws, u, which='p', int8_projection=int8, use_graph=True, **kw)
            assert torch.equal(h, hyp) and torch.equal(s, score)
            eng.greedy_decode(ws, which='p')             # eager work of the program between the replays
            torch.cuda.synchronize()
    assert sum(k[0] == 'sample' for k in ws['graph'] if isinstance(k, tuple)) == 1


def test_ema_and_p_weights_do_not_mix():
    eng, ws = network('small_dropout')
    L, B = ws['L'], ws['B']
    u = uniforms(L, B)
    eng.store.ema.mul_(0.5)
    want = {}
    for which in ('p', 'ema', 'p', 'ema'):
        eng.sample_decode(ws, u, which=which, int8_projection=True)
        out = ws['proj']['out'].clone()
        assert torch.equal(want.setdefault(which, out), out)
    assert not torch.equal(want['p'], want['ema'])


def test_refusals():
    eng, ws = network('tiny_odd')
    L, B = ws['L'], ws['B']
    u = uniforms(L, B)
    for bad in (u.double(), u[:, :-1], u[:-1], u.cpu(), u.reshape(-1), None):
        with pytest.raises(ValueError):
            eng.sample_decode(ws, bad, which='p')
    for kw in (dict(temperature=torch.ones(B + 1, device='cuda')), dict(top_k=torch.ones(B, dtype=torch.int32)), dict(top_p=torch.ones(B, 1, device='cuda'))):
        with pytest.raises(ValueError):
            eng.sample_decode(ws, u, which='p', **kw)


def test_online_predictor_draws(tmp_path, monkeypatch):
    """The predictor of a trained model with `sampling`: temperature 0 gives its greedy words, a seed repeats its drawn ones, an utterance
    alone works like a batch."""
    import os
    from ecog2txt_amd.data_generators import ECoGDataGenerator, SyntheticSpeechDataGenerator
    from ecog2txt_amd.trainers import MultiSubjectTrainer
    from experiment_fixture import make_experiment
    monkeypatch.setattr(ECoGDataGenerator, 'text_dir', str(tmp_path))
    for k, v in dict(num_sentences=6, trials_per_block=24, max_words=5).items():
        monkeypatch.setattr(SyntheticSpeechDataGenerator, k, v)
    path = make_experiment(tmp_path, subject_ids=(401,), epochs=2, interval=2)
    ck = str(tmp_path / 'ck')
    os.makedirs(ck)
    tr = MultiSubjectTrainer(path, [401], checkpoint_dir=ck, VERBOSE=False, SN_kwargs={'N_cases': 32, 'EMA_decay': 0.9}, DG_kwargs={'max_samples': 420})
    for s in tr.ecog_subjects:
        s.write_tf_records_maybe()
    tr.parallel_transfer_learn()
    X = tr.net._stage(tr.ecog_subjects[-1], 'validation')['X'][:5]
    greedy = tr.construct_online_predictor()(X)
    assert tr.construct_online_predictor(sampling=dict(temperature=0.0))(X) == greedy
    kw = dict(temperature=1.2, top_k=20, top_p=0.98, int8_projection=True)
    one, two, other = (tr.construct_online_predictor(sampling=dict(kw, seed=n)) for n in (7, 7, 8))
    a, b = [one(X), one(X)], [two(X), two(X)]
    assert a == b and a[0] != a[1] and a[0] != other(X)              # (24 and more drawn words: equal by chance once in thousands)
    assert len(one(X[0])) == 1
    with pytest.raises(ValueError):
        tr.construct_online_predictor(sampling=dict(topk=3))
