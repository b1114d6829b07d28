"""A file's 4-bit microscaled tensors: listed with their bytes (no GPU), and laid out for the products (GPU)."""
import numpy as np
import pytest

from helpers import write_gguf


def _file(tmp_path, rows, k, seed=3):
    rng = np.random.RandomState(seed)
    blocks = rng.randint(0, 256, (rows, k // 32, 17)).astype(np.uint8)
    blocks[:, :, 0] = rng.randint(118, 126, (rows, k // 32))
    path = str(tmp_path / "m.gguf")
    write_gguf(path, [("general.architecture", "str", "any")], [("blk.0.w", 39, [k, rows], blocks.tobytes())])
    return path, blocks


def test_listed_with_their_bytes(tmp_path):
    from denno_beta_b200 import gguf

    path, blocks = _file(tmp_path, 5, 96)
    with gguf.GgufFile(path) as g:
        info = g.tensor("blk.0.w")
        assert info["type"] == 39 and info["dims"] == [96, 5] and info["nbytes"] == 5 * 3 * 17
        assert g.tensor_bytes("blk.0.w").tobytes() == blocks.tobytes()


@pytest.mark.gpu
def test_from_a_file_to_a_product(tmp_path):
    import torch

    import dense_helpers as dh
    from denno_beta_b200 import cuda as cu, gguf

    rows, k, nt = 200, 352, 9
    path, blocks = _file(tmp_path, rows, k)
    c = cu.CudaCtx(0)
    try:
        c.set_stream(1)
        with gguf.GgufFile(path) as g:
            raw = torch.from_numpy(np.array(g.tensor_bytes("blk.0.w"))).cuda()
        codes, scales = (torch.empty(n, dtype=torch.uint8, device="cuda") for n in cu.mx4_bytes(rows, k))
        assert c.mx4_quantize_dev(cu.MXFP4, raw.data_ptr(), rows, k, codes.data_ptr(), scales.data_ptr())
        x = torch.randn(nt, k, generator=torch.Generator().manual_seed(1))
        xc, xs = (torch.empty(n, dtype=torch.uint8, device="cuda") for n in cu.mx4_bytes(nt, k))
        dev, out = x.cuda(), torch.empty(nt, rows, device="cuda")
        assert c.mx4_quantize_dev(cu.F32, dev.data_ptr(), nt, k, xc.data_ptr(), xs.data_ptr())
        assert c.mx4_gemm_dev(xc.data_ptr(), xs.data_ptr(), codes.data_ptr(), scales.data_ptr(), nt, k, rows, cu.F32, out.data_ptr())
        torch.cuda.synchronize()
        b = torch.from_numpy(blocks)
        w = dh.values(torch.cat([b[:, :, 1:] & 15, b[:, :, 1:] >> 4], -1).reshape(rows, k), b[:, :, 0])
        vx = dh.values(*dh.quantise(x))
        assert bool(((out.cpu().double() - vx @ w.T).abs() <= dh.sum_error(k, vx.abs() @ w.abs().T)).all())
        # its blocks are no type of a registered matrix or expert: those calls decline and write nothing
        assert not c.register_matrix(1, cu.MXFP4, blocks.reshape(-1), k, rows)
        assert not c.gemv_dev(cu.MXFP4, raw.data_ptr(), k, rows, dev.data_ptr(), out.data_ptr())
        assert c.device_status() == 0
    finally:
        c.close()
