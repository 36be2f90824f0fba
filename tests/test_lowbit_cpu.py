"""8-bit operators, what can be checked without a GPU: struct layouts and refusals of the C entry points, refusals of the Python
ones, and the oracle itself against independent statements of the formats."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest
import torch

from conv1d_text_vae_amd import _lib as L
from oracle import lowbit_oracle as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_sizes_and_constants_match_the_header(tmp_path):
    structs = {'c1v_fp8_quant_args': L.Fp8QuantArgs, 'c1v_fp8_gemm_args': L.Fp8GemmArgs, 'c1v_fp8_dense_args': L.Fp8DenseArgs,
               'c1v_fp8_linear_args': L.Fp8LinearArgs, 'c1v_adamw_tensor': L.AdamwTensor, 'c1v_adamw_args': L.AdamwArgs}
    consts = {'C1V_FP8_BLOCK': L.FP8_BLOCK, 'C1V_FP8_ROWS': L.FP8_ROWS, 'C1V_ADAMW_CHUNK': L.ADAMW_CHUNK,
              'C1V_ADAMW_GROUP': L.ADAMW_GROUP, 'C1V_ADAMW_PARTIALS': L.ADAMW_PARTIALS}
    src = '#include <stdio.h>\n#include "c1dvae.h"\nint main(void){\n'
    src += ''.join('printf("%s %%zu\\n", sizeof(%s));' % (s, s) for s in structs)
    src += ''.join('printf("%s %%d\\n", %s);' % (s, s) for s in consts) + 'return 0;}\n'
    (tmp_path / 's.c').write_text(src)
    subprocess.check_call(['gcc', '-I', os.path.join(ROOT, 'include'), str(tmp_path / 's.c'), '-o', str(tmp_path / 's')])
    got = dict(line.split() for line in subprocess.check_output([str(tmp_path / 's')]).decode().splitlines())
    assert {k: int(v) for k, v in got.items()} == {**{k: C.sizeof(v) for k, v in structs.items()}, **consts}


def test_packed_argument_structs_have_the_mirrors_layouts():
    """fp8.py passes the structs as packed bytes: every field of a sample lands where the ctypes mirror has it."""
    from conv1d_text_vae_amd import fp8

    def flat(cls, v):
        out = []
        for name, kind in cls._fields_:
            x = getattr(v, name)
            out += flat(kind, x) if issubclass(kind, C.Structure) else [x or 0]
        return out
    for pack, cls in ((fp8._QUANT, L.Fp8QuantArgs), (fp8._PRODUCT, L.Fp8GemmArgs), (fp8._DENSE, L.Fp8DenseArgs), (fp8._LINEAR, L.Fp8LinearArgs)):
        n = len(flat(cls, cls()))
        data = pack(*range(1, n + 1))
        # (trailing padding of a struct is not packed; the library does not read it)
        assert C.sizeof(cls) - 8 < len(data) <= C.sizeof(cls), cls
        v = cls.from_buffer_copy(data.ljust(C.sizeof(cls), b'\0'))
        assert flat(cls, v) == list(range(1, n + 1)), cls


def test_c_entry_points_refuse_on_the_host():
    """Nothing here launches: every call is refused before, with a message."""
    lib = L.load()
    mem = (C.c_char * 8192)()
    p = (C.addressof(mem) + 255) & ~255

    def refused(fn, args, text):
        assert getattr(lib, fn)(None if args is None else C.byref(args), None) != 0
        assert text in lib.c1v_last_error(), (fn, lib.c1v_last_error())

    refused('c1v_fp8_quantize', None, b'null')
    q = dict(x=p, dtype=0, rows=4, cols=8, ld=8, q=p, s=p)
    for change, text in ((dict(x=None), b'null'), (dict(dtype=2), b'dtype'), (dict(rows=0), b'shape'), (dict(ld=7), b'shape'), (dict(s=None), b'together'),
                         (dict(q=None, s=None), b'together'), (dict(q=p + 8), b'aligned'), (dict(colsum=p), b'colsum'), (dict(cols=1 << 23, ld=1 << 23), b'large'), (dict(rows=1 << 28), b'large'),
                         (dict(rows=1 << 27, cols=1 << 22, ld=1 << 22), b'large')):
        refused('c1v_fp8_quantize', L.Fp8QuantArgs(**{**q, **change}), text)
    g = dict(a=p, sa=p, b=p, sb=p, m=64, n=64, kp=128, out_dtype=0, out=p, ldo=64)
    for change, text in ((dict(a=None), b'null'), (dict(m=0), b'shape'), (dict(kp=100), b'whole blocks'), (dict(out_dtype=3), b'out_dtype'),
                         (dict(ldo=63), b'ldo'), (dict(b=p + 4), b'aligned'), (dict(kp=8192), b'workspace'), (dict(m=1 << 31), b'large')):
        refused('c1v_fp8_gemm', L.Fp8GemmArgs(**{**g, **change}), text)
    ok = L.Fp8GemmArgs(**{**g, 'm': 4})
    for change, text in ((dict(x=None), b'null'), (dict(x_dtype=5), b'x_dtype'), (dict(k=129), b'shape'), (dict(ldx=100), b'shape')):
        refused('c1v_fp8_dense', L.Fp8DenseArgs(**{**dict(x=p, x_dtype=0, ldx=128, k=128, g=ok), **change}), text)
    assert [lib.c1v_fp8_dense_direct(*s) for s in ((16, 1 << 20, 1 << 20), (256, 512, 1920), (1024, 1024, 384), (32, 64, 2176))] == [1, 1, 0, 0]
    refused('c1v_fp8_dense', L.Fp8DenseArgs(x=p, x_dtype=0, ldx=128, k=128, g=L.Fp8GemmArgs(**{**g, 'm': 1024, 'n': 1024, 'ldo': 1024, 'a': None, 'sa': None})), b'room')
    lin = dict(rows=4, k=8, n=8, need_dx=1, need_dk=1, need_db=1)
    refused('c1v_fp8_linear_fwd', L.Fp8LinearArgs(**lin), b'null')
    refused('c1v_fp8_linear_bwd', L.Fp8LinearArgs(**lin), b'null')
    refused('c1v_fp8_linear_fwd', L.Fp8LinearArgs(**{**lin, 'k': 0}), b'shape')
    refused('c1v_fp8_linear_fwd', L.Fp8LinearArgs(**{**lin, 'rows': 1 << 24}), b'rows')         # before the backward pass would
    refused('c1v_fp8_linear_fwd', L.Fp8LinearArgs(**{**lin, 'n': (1 << 22) + 1}), b'large')
    refused('c1v_fp8_dense', L.Fp8DenseArgs(x=p, x_dtype=0, ldx=128, k=128, g=L.Fp8GemmArgs(**{**g, 'm': 4, 'n': 1 << 27, 'ldo': 1 << 27})), b'shape')
    refused('c1v_fp8_linear_bwd', L.Fp8LinearArgs(**{**lin, 'dy': p, 'keep': p, 'temp': p}), b'gradient')
    refused('c1v_fp8_linear_bwd', L.Fp8LinearArgs(**{**lin, 'dy': p, 'keep': p + 4, 'temp': p}), b'aligned')
    assert lib.c1v_fp8_linear_sizes(None, None, None, None) != 0
    w = dict(tensors=p, host=p, p=p, g=p, m=p, v=p, t=p, lr=p, sched=p, norm=p, p_dtype=p, g_dtype=p, n_tensors=1, beta1=0.9, beta2=0.99, eps=1e-8)
    refused('c1v_adamw_step', None, b'null')
    for change, text in ((dict(t=None), b'null'), (dict(p_dtype=None), b'null'), (dict(n_tensors=0), b'count'), (dict(states=2), b'states'), (dict(states=1), b'scales'),
                         (dict(m=p + 4), b'aligned'), (dict(beta1=1.0), b'betas'), (dict(eps=0.0), b'eps'), (dict(clipnorm=1.0), b'partial sums')):
        refused('c1v_adamw_step', L.AdamwArgs(**{**w, **change}), text)
    table, ptr, kind = (L.AdamwTensor * 2)(L.AdamwTensor(10, 0, 0.0, 0), L.AdamwTensor(10, 128, 0.0, 1)), (C.c_void_p * 2)(p, None), (C.c_uint8 * 2)(0, 0)
    w = dict(w, n_tensors=2, host=C.addressof(table), p=C.addressof(ptr), g=C.addressof(ptr), p_dtype=C.addressof(kind), g_dtype=C.addressof(kind))
    refused('c1v_adamw_step', L.AdamwArgs(**w), b'tensor 1 has no parameter')
    ptr[1], kind[1] = p, 7
    refused('c1v_adamw_step', L.AdamwArgs(**w), b'dtype of tensor 1')
    kind[1] = 0
    for bad in (L.AdamwTensor(10, 100, 0.0, 1), L.AdamwTensor(10, 128, 0.0, 2), L.AdamwTensor(-1, 128, 0.0, 1)):
        table[1] = bad
        refused('c1v_adamw_step', L.AdamwArgs(**w), b'table entry 1')


def test_sizes_of_workspaces():
    lib = L.load()
    k, f, b = (C.c_int64() for _ in range(3))
    a = L.Fp8LinearArgs(rows=300, k=200, n=100, need_dx=1, need_dk=1, need_db=1)
    assert lib.c1v_fp8_linear_sizes(C.byref(a), C.byref(k), C.byref(f), C.byref(b)) == 0
    assert k.value >= 200 * 128 + 208 + 200 * 384 + 3 * 208               # kernel and x, values and scales
    assert f.value >= 300 * 256 + 2 * 304 + 100 * 256 + 2 * 112
    assert b.value >= 300 * 128 + 304 + 100 * 384 + 3 * 112 + 3 * 100 * 4
    a = L.Fp8LinearArgs(rows=300, k=200, n=100)
    assert lib.c1v_fp8_linear_sizes(C.byref(a), C.byref(k), C.byref(f), C.byref(b)) == 0 and k.value == 0
    assert lib.c1v_fp8_gemm_work(512, 512, 8192) == 4 * 512 * 512 * 4 or lib.c1v_fp8_gemm_work(512, 512, 8192) % (512 * 512 * 4) == 0
    assert lib.c1v_fp8_gemm_work(8192, 8192, 8192) == 0


def test_python_refuses_without_a_gpu():
    from conv1d_text_vae_amd import fp8, optim
    from conv1d_text_vae_amd.seq2seq import Seq2SeqGenerator
    x = torch.zeros(4, 130)
    w = fp8.Fp8Rows(torch.zeros(8, 256).to(torch.float8_e4m3fn), torch.full((2, 16), 127, dtype=torch.uint8), 130)
    assert w.rows == 8 and w.dequantize().shape == (8, 130)
    for f in (lambda: fp8.quantize_rows(x), lambda: fp8.quantize_both(x), lambda: fp8.dense(x, w), lambda: fp8.product(w, w),
              lambda: fp8.linear(x, torch.zeros(130, 4)), lambda: optim.AdamW([x]),
              # (a generator can be made anywhere, to hold loaded weights; it refuses to compute)
              lambda: Seq2SeqGenerator(4, 3, 5, 6, device='cpu', products='fp8').encode(torch.ones(2, 4, 3)),
              lambda: Seq2SeqGenerator(4, 3, 5, 6, device='cpu', products='fp8').eval_batch(torch.ones(2, 4, 3), torch.ones(2, 4, 5), torch.ones(2, 4, 5)),
              lambda: Seq2SeqGenerator(4, 3, 5, 6, device='cpu', optimizer='adamw8').train_batch(torch.ones(2, 4, 3), torch.ones(2, 4, 5), torch.ones(2, 4, 5))):
        with pytest.raises(L.C1VError):
            f()
    for f in (lambda: fp8.quantize_rows(x.double()), lambda: fp8.quantize_rows(x[0]), lambda: fp8.quantize_rows(x[:, :0]),
              lambda: fp8.Fp8Rows(w.data, w.scale, 129 + 128), lambda: fp8.Fp8Rows(w.data, w.scale.t(), 130), lambda: fp8.Fp8Rows(x, w.scale, 130),
              lambda: fp8.linear(x, torch.zeros(131, 4)), lambda: fp8.linear(x, torch.zeros(130, 4), torch.zeros(5)), lambda: optim.AdamW([x], states='16bit'),
              lambda: optim.AdamW([x, x + 1], weight_decay=[0.1, float('nan')]), lambda: optim.AdamW([x], lr=float('inf')),
              lambda: optim.AdamW([x], lr=float('nan')), lambda: optim.AdamW([x], clipnorm=float('nan')), lambda: optim.AdamW([x], eps=float('inf')),
              lambda: Seq2SeqGenerator(4, 3, 5, 6, device='cpu', products='int8'), lambda: Seq2SeqGenerator(4, 3, 5, 6, device='cpu', optimizer='sgd')):
        with pytest.raises(ValueError):
            f()


def test_operands_at_any_strides():
    """Values and scales as a transposition or a slice leaves them (scales made row by row and transposed, when the number of
    rows needs no padding, are such)."""
    from conv1d_text_vae_amd import fp8
    data = torch.arange(32 * 256).remainder(97).float().view(32, 256).to(torch.float8_e4m3fn)
    scale = (torch.arange(2 * 32) + 100).to(torch.uint8).view(2, 32)
    want = fp8.Fp8Rows(data, scale, 200)
    wide = torch.zeros(32, 300, dtype=torch.uint8)
    wide[:, :256] = data.view(torch.uint8)
    values, turned = wide.view(torch.float8_e4m3fn)[:, :256], scale.t().contiguous().t()
    assert not values.is_contiguous() and not turned.is_contiguous()
    for q in (fp8.Fp8Rows(data, turned, 200), fp8.Fp8Rows(values, scale, 200), fp8.Fp8Rows(values, turned, 200)):
        assert q.data.is_contiguous() and q.scale.is_contiguous() and torch.equal(q.scale, scale)
        assert torch.equal(q.dequantize(), want.dequantize())
    assert want.data is data and want.scale is scale                      # nothing is copied that needs no copy


def test_generator_defaults_are_the_reference_ones():
    from conv1d_text_vae_amd import Conv1dTextVAE
    from conv1d_text_vae_amd.seq2seq import Seq2SeqGenerator
    g = Seq2SeqGenerator(4, 3, 5, 6, device='cpu')
    assert (g.optimizer, g.products, g.opt) == ('rmsprop', 'f32', None)
    assert (Conv1dTextVAE.vae_optimizer, Conv1dTextVAE.generator_optimizer, Conv1dTextVAE.generator_products) == ('nadam', 'rmsprop', 'f32')


def test_the_largest_number_of_rows_fits_a_launch():
    """2^28 - 16 rows are 2^24 - 1 workgroups of 256 threads; one more row would be 2^32 threads, which no launch takes."""
    lib = L.load()
    mem = (C.c_char * 4096)()
    p = (C.addressof(mem) + 255) & ~255
    for rows in ((1 << 28) - 15, (1 << 28) - 1):
        assert lib.c1v_fp8_quantize(C.byref(L.Fp8QuantArgs(x=p, dtype=0, rows=rows, cols=8, ld=8, q=p, s=p)), None) != 0
        assert b'large' in lib.c1v_last_error()
        a = L.Fp8LinearArgs(rows=rows, k=8, n=8, need_dx=1)
        assert lib.c1v_fp8_linear_sizes(C.byref(a), *(C.byref(C.c_int64()) for _ in range(3))) != 0 and b'rows' in lib.c1v_last_error()
    a = L.Fp8LinearArgs(rows=(1 << 28) - 16, k=8, n=8, need_dx=1)
    assert lib.c1v_fp8_linear_sizes(C.byref(a), *(C.byref(C.c_int64()) for _ in range(3))) == 0


def test_workspace_of_a_k_in_runs():
    """Partial sums [runs][m][n rounded up to 4] in fp32, exactly: from 32 blocks of K four runs up to 64 tiles of 64 x 64 and two
    up to 128 tiles, none for more tiles, a shorter K or the larger tiles."""
    work = L.load().c1v_fp8_gemm_work
    for m, n, blocks, runs in ((512, 512, 64, 4), (512, 512, 32, 4), (512, 512, 31, 1), (66, 130, 34, 4), (1, 1, 32, 4), (64 * 64, 64, 32, 4), (64 * 64 + 1, 64, 31, 1),
                               (64 * 64 + 1, 64, 32, 2), (512, 1024, 32, 2), (512, 1021, 33, 2), (512, 1025, 64, 1), (768, 1024, 64, 1), (8192, 8192, 64, 1)):
        assert work(m, n, 128 * blocks) == (runs * m * (-(-n // 4) * 4) * 4 if runs > 1 else 0), (m, n, blocks)


def test_an_operand_without_rows_or_columns():
    from conv1d_text_vae_amd import fp8
    e4 = lambda *s: torch.zeros(s, dtype=torch.uint8).view(torch.float8_e4m3fn)
    assert fp8.Fp8Rows(e4(0, 256), torch.zeros(2, 0, dtype=torch.uint8), 130).dequantize().shape == (0, 130)
    assert fp8.Fp8Rows(e4(5, 0), torch.zeros(0, 16, dtype=torch.uint8), 0).dequantize().shape == (5, 0)


def test_one_weight_decay_of_any_number_type():
    from conv1d_text_vae_amd import optim
    for wd in (0.1, 1, np.float32(0.1), np.float64(0.1), np.int64(1)):
        with pytest.raises(L.C1VError):                                   # (taken, and then no GPU)
            optim.AdamW([torch.zeros(3), torch.zeros(2)], weight_decay=wd)
    for wd in (np.float32('nan'), np.float32(-1), [np.float32(0.1)]):
        with pytest.raises(ValueError):
            optim.AdamW([torch.zeros(3), torch.zeros(2)], weight_decay=wd)


def test_products_without_a_gradient_are_refused_where_one_is_asked_for():
    from conv1d_text_vae_amd import fp8
    x, b = torch.zeros(4, 130), torch.zeros(8)
    w = fp8.Fp8Rows(torch.zeros(8, 256).to(torch.float8_e4m3fn), torch.full((2, 16), 127, dtype=torch.uint8), 130)
    xg, bg = x.clone().requires_grad_(True), b.clone().requires_grad_(True)
    calls = (lambda: fp8.dense(xg, w), lambda: fp8.dense(x, w, bg), lambda: fp8.product(w, w, bg))
    for f in calls:
        with pytest.raises(ValueError, match='gradient'):
            f()
        with torch.no_grad(), pytest.raises(L.C1VError):                  # (and then for want of a GPU)
            f()


def test_estimator_keeps_its_choices_when_pickled():
    """Unfitted and fitted; a fitted one serves as it was fitted, whatever was chosen since; states of before load as they did."""
    import copy
    import pickle
    from conv1d_text_vae_amd import Conv1dTextVAE
    from conv1d_text_vae_amd import estimator as E
    from conv1d_text_vae_amd.embeddings import synthetic_fasttext
    emb = synthetic_fasttext(['aa', 'bb'], vector_size=6, bucket=20, seed=1)
    choices = lambda v: (v.vae_optimizer, v.generator_optimizer, v.generator_products)
    vae = Conv1dTextVAE(emb, emb, n_filters=4, latent_dim=3, n_recurrent_units=5)
    assert 'vae_optimizer' not in pickle.loads(pickle.dumps(vae)).get_params() and choices(pickle.loads(pickle.dumps(vae))) == choices(Conv1dTextVAE)
    vae.vae_optimizer, vae.generator_optimizer, vae.generator_products = 'adamw8', 'adamw', 'fp8'
    for other in (pickle.loads(pickle.dumps(vae)), copy.deepcopy(vae)):
        assert choices(other) == ('adamw8', 'adamw', 'fp8')
    vae.input_text_size_ = vae.output_text_size_ = 4
    vae.input_vector_size_ = vae.output_vector_size_ = 8
    vae.output_text_size_in_characters_, vae.target_char_index_, vae.reverse_target_char_index_ = 9, {'a': 0, 'b': 1}, {0: 'a', 1: 'b'}
    rt, gen = vae._create_model(8, 8, seed=1)
    vae._vae_runtime, vae._generator = rt, gen
    vae.vae_encoder_, vae.vae_decoder_ = E.VAEEncoderModel(rt), E.VAEDecoderModel(rt)
    vae.generator_encoder_, vae.generator_decoder_ = gen.encoder_model(), gen.decoder_model()
    got = pickle.loads(pickle.dumps(vae))
    assert choices(got) == ('adamw8', 'adamw', 'fp8')
    assert (got._generator.products, got._generator.optimizer, got._vae_runtime.optimizer) == ('fp8', 'adamw', 'adamw8')
    assert all(np.array_equal(v, got._generator.get_weights()[k]) for k, v in gen.get_weights().items())
    vae.generator_products = 'f32'
    got = pickle.loads(pickle.dumps(vae))
    assert got.generator_products == 'f32' and got._generator.products == 'fp8'
    old = {k: v for k, v in vae.__getstate__().items() if not k.endswith('_optimizer') and not k.startswith('generator_products')}
    got = Conv1dTextVAE.__new__(Conv1dTextVAE)
    got.__setstate__(old)
    assert choices(got) == choices(Conv1dTextVAE) and got._generator.products == 'f32'


# ---------------------------------------------------------------------------------------------------------------
# the oracle
# ---------------------------------------------------------------------------------------------------------------
def test_oracle_rounds_to_e4m3_as_the_type_does():
    u = np.concatenate([np.linspace(-448, 448, 20001), 2.0 ** np.linspace(-14, 8.8, 4001), [0.0, 2.0 ** -10, 3 * 2.0 ** -10]]).astype(np.float32)
    want = torch.from_numpy(u).to(torch.float8_e4m3fn)
    np.testing.assert_array_equal(O.e4m3_nearest(u), want.float().numpy())
    np.testing.assert_array_equal(O.e4m3_values(want.view(torch.uint8).numpy()), want.float().numpy())


def test_oracle_scales():
    x = np.zeros((4, 130))
    x[0, 0], x[1, 5], x[2, 129], x[3, 7] = 448.0, -449.0, 1e-3, np.inf
    q, e = O.quantize(x)
    assert e.tolist() == [[0, 0], [1, 0], [0, -18], [0, 0]]      # 1e-3 / 448 = 2.2e-6 <= 2^-18
    assert np.isnan(q[3, 7]) and np.isnan(q).sum() == 1
    np.testing.assert_array_equal(O.values(q, e)[0, 0], 448.0)


def test_oracle_random_bits_are_philox():
    from oracle.vae_oracle import philox4x32
    h = O.halves(24, (5 << 32) + 9, 3)
    w = philox4x32(np.array([[2, 0, 3, 0]], dtype=np.uint32), (9, 5))[0].astype(np.int64)
    assert h[16:].tolist() == [x for v in w for x in (v & 0xFFFF, v >> 16)]


def test_oracle_states_are_rounded_to_a_neighbour_and_in_the_mean():
    """Every random number of 16 bits once: the value lies between the two codes taken, which are neighbours, and their mean is
    the value up to 2^-16 of a step (and the 2^-20 that the definition cuts)."""
    r = np.arange(65536)
    for x in (1.0, 1.03, -0.77, 3.1e-5, -2.9e-4, 0.0):
        m = np.full(65536, x, dtype=np.float32)
        m[::128] = 1.2                                           # the block's largest value sets the scale
        got = O.unpack_m(*O.pack_m(m, r))
        keep = np.arange(65536) % 128 != 0
        lo, hi = got[keep].min(), got[keep].max()
        assert lo <= x * (1 + 1e-6) + 1e-12 or x < 0
        assert len(np.unique(got[keep])) <= 2 and lo - 1e-9 <= np.float32(x) <= hi + 1e-9
        assert abs(got[keep].mean() - np.float32(x)) <= (hi - lo) * 2.0 ** -7 + 1e-12      # 1/128 of the numbers left out
    for x in (1.0, 1.9, 0.013, 7e-8, 0.0):
        v = np.full(65536, x, dtype=np.float32)
        v[::128] = 2.0
        code, s = O.pack_v(v, r)
        got = O.unpack_v(code, s)[np.arange(65536) % 128 != 0]
        assert len(np.unique(got)) <= 2 and got.min() <= np.float32(x) <= got.max()
        assert abs(got.mean() - np.float32(x)) <= (got.max() - got.min()) * 2.0 ** -7 + 1e-12
    code, s = O.pack_v(np.r_[np.full(127, 1e-30), 1.0].astype(np.float32), np.zeros(128, dtype=np.int64))
    assert (code[:127] == 1).all() and (O.unpack_v(code, s)[:127] > 0).all()      # never zero
    code, s = O.pack_v(np.r_[np.zeros(126), np.nan, np.inf].astype(np.float32), np.zeros(128, dtype=np.int64))
    assert code.tolist() == [0] * 126 + [255, 255]


def test_oracle_adamw_first_step_is_the_sign():
    p, m, v = O.adamw(np.ones(3), np.array([2.0, -0.5, 0.0]), 0.0, 0.0, 1, 0.1, 0.9, 0.999, 0.0 + 1e-30, 0.5, 1.0)
    np.testing.assert_allclose(p, 0.95 - 0.1 * np.array([1.0, -1.0, 0.0]))
    f, n = O.clip_factor([np.array([3.0]), np.array([4.0])], 1.0)
    assert n == 5.0 and f == 0.2 and O.clip_factor([np.array([3.0])], 0.0)[0] == 1.0
