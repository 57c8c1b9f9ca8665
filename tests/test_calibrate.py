"""gpuq/calibrate.py: a layer's Hessians from its rows, logits and stored MXFP4 experts against numpy in 64 bits, the
folder that requant.py reads, and what it refuses.

Tolerances: H_in sums exact products of the rows themselves (f64: 1e-12). The hidden rows come from f32 sums of ne0 terms
and SwiGLU, within 4 (ne0 + 8) 2^-23 of sum |x w| as the products' own tests derive, so a pair's product is within twice
that of the rows' sizes; H_mid is held to 1e-3 of the largest entry of its diagonal, above that for these sizes."""
import os

import numpy as np
import pytest

from gpuq import calibrate, gguf_io, requant

T = gguf_io.TYPE_BY_NAME
LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def stored(rng, nexp, nff, ne0):
    """(blocks [nexp, nff, ne0 / 32 * 17], their values in f64)"""
    code = rng.integers(0, 16, (nexp, nff, ne0 // 32, 2, 16)).astype(np.uint8)
    e = rng.integers(119, 124, (nexp, nff, ne0 // 32, 1)).astype(np.uint8)
    blocks = np.concatenate((e, code[..., 0, :] | (code[..., 1, :] << 4)), axis=-1)
    v = LEVELS[code & 7] * np.where(code & 8, -1.0, 1.0)
    v = v.reshape(nexp, nff, ne0 // 32, 32) * np.exp2(e.astype(np.float64) - 127)
    return blocks.reshape(nexp, nff, -1), v.reshape(nexp, nff, ne0)


def model_file(path, gate, up, nexp, nff, ne0, ttype="MXFP4"):
    with gguf_io.GGUFWriter(path) as w:
        w.add_tensor_info("blk.3.ffn_gate_exps.weight", (ne0, nff, nexp), T[ttype])
        w.add_tensor_info("blk.3.ffn_up_exps.weight", (ne0, nff, nexp), T[ttype])
        w.write_header()
        w.write_tensor_data(gate)
        w.write_tensor_data(up)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_hessians_of_a_layer(tmp_path, dtype):
    import torch
    torch.cuda.init()
    import gpuq
    gq = gpuq.load_gpuq(0)
    rng = np.random.default_rng(1)
    nexp, nff, ne0, n, topk = 6, 256, 512, 333, 2
    gate, gv = stored(rng, nexp, nff, ne0)
    up, uv = stored(rng, nexp, nff, ne0)
    x = (0.1 * rng.standard_normal((n, ne0))).astype(dtype)
    logits = rng.permuted(np.tile(np.arange(nexp) * 0.5, (n, 1)), axis=1).astype(np.float32)
    logits[:, 4] = -np.inf                               # an expert that nothing reaches
    model = str(tmp_path / "m.gguf")
    model_file(model, gate, up, nexp, nff, ne0)
    np.save(tmp_path / "blk.3.x.npy", x)
    np.save(tmp_path / "blk.3.logits.npy", logits)
    out = str(tmp_path / "hess")
    calibrate.run(model, 3, str(tmp_path), out, topk, gq=gq, chunk=100)
    ids = np.argsort(-logits, axis=1, kind="stable")[:, :topk]
    hin, hmid = np.load(os.path.join(out, "blk.3.in.npy")), np.load(os.path.join(out, "blk.3.mid.npy"))
    counts = np.load(os.path.join(out, "blk.3.counts.npy"))
    assert counts.tolist() == [int((ids == e).sum()) for e in range(nexp)] and counts[4] == 0
    for e in range(nexp):
        xe = x[(ids == e).any(axis=1)].astype(np.float64)
        want = xe.T @ xe
        assert np.abs(hin[e] - want).max() <= 1e-12 * max(1.0, np.abs(want).max())
        g = xe @ gv[e].T
        mid = g / (1 + np.exp(-g)) * (xe @ uv[e].T)
        want = mid.T @ mid
        assert np.abs(hmid[e] - want).max() <= 1e-3 * max(np.abs(want).max(), 1e-300)
    assert requant.hess_file(out, "blk.3.ffn_gate_exps.weight") == (os.path.join(out, "blk.3.in.npy"),
                                                                    os.path.join(out, "blk.3.counts.npy"))
    assert requant.hess_file(out, "blk.3.ffn_down_exps.weight")[0] == os.path.join(out, "blk.3.mid.npy")


@pytest.mark.gpu
def test_an_expert_rounds_with_its_hessian():
    """the whole path: a layer's own Hessian, its factor and the feedback loop lower the calibration rows' error"""
    import torch
    torch.cuda.init()
    import gpuq
    from gpuq import ldlq
    gq = gpuq.load_gpuq(0)
    rng = np.random.default_rng(2)
    nexp, nff, ne0 = 2, 256, 512
    gate, gv = stored(rng, nexp, nff, ne0)
    up, _ = stored(rng, nexp, nff, ne0)
    h = calibrate.ExpertHessians(gq, torch.from_numpy(gate).cuda(), torch.from_numpy(up).cuda(), nexp, nff, ne0, 1)
    mix = rng.standard_normal((ne0, ne0)) / np.sqrt(ne0)
    x = torch.from_numpy((0.1 * rng.standard_normal((2000, ne0)) @ (np.eye(ne0) + 2 * mix)).astype(np.float32)).cuda()
    h.add(x, torch.from_numpy(rng.standard_normal((2000, nexp)).astype(np.float32)).cuda())
    H, n = h.hin[0].cpu().numpy(), int(h.counts[0])
    U, perm, diag_n, _ = ldlq.prepare_hessian_torch(h.hin[0], n)
    W = torch.from_numpy(gv[:1].astype(np.float32)).cuda()
    qw = torch.from_numpy(ldlq.block_weights("diag", diag_n=diag_n)[None]).cuda()
    loss = []
    for feedback in (False, True):
        q = ldlq.quantize_matrix_dev(gq, gpuq.Q2_K, W, U, perm, qw, feedback=feedback)
        deq = torch.empty(nff, ne0, device="cuda")
        assert gq.gpuq_dequantize_dev(gpuq.Q2_K, q.data_ptr(), deq.data_ptr(), nff * ne0 // 256,
                                      torch.cuda.current_stream().cuda_stream)
        loss.append(ldlq.proxy_loss(gv[0], deq.cpu().numpy(), H, n))
    assert loss[1] < loss[0]


def test_refusals(tmp_path):
    model = str(tmp_path / "m.gguf")
    model_file(model, np.zeros((2, 256, 256), np.float32), np.zeros((2, 256, 256), np.float32), 2, 256, 256, "F32")
    with pytest.raises(ValueError, match="not MXFP4"):
        calibrate.run(model, 3, str(tmp_path), str(tmp_path), 1, gq=object())
    with pytest.raises(ValueError, match="whole 256s"):
        calibrate.ExpertHessians(None, None, None, 2, 100, 256, 1)
    assert calibrate.main(["a", "b"]) == 2 and calibrate.main(["m", "0", "r", "o", "--topk=1", "--what=2"]) == 2
