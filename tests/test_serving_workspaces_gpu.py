"""Workspaces that the serving operators refuse (B200 only)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def kernels():
    from trinity_lowering import kernels as k
    k.library()
    return k


def decode(kernels, heads=8, workspace=None):
    cache = kernels.kv4_cache(4, 2, 32, 128, 64, DEV)
    q = torch.zeros(2, heads, 128, dtype=BF16, device=DEV)
    table = torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    return kernels.kv4_decode(q, cache, table, torch.ones(2, dtype=torch.int32, device=DEV), 1.0, workspace=workspace)


def project(kernels, rank=16, workspace=None):
    x = torch.zeros(4, 64, dtype=BF16, device=DEV)
    w = torch.zeros(64, 64, dtype=BF16, device=DEV)
    down, up = torch.zeros(2, 64, rank, dtype=BF16, device=DEV), torch.zeros(2, rank, 64, dtype=BF16, device=DEV)
    return kernels.gemm_adapters(x, w, down, up, torch.zeros(4, dtype=torch.int32, device=DEV), workspace=workspace)


def test_a_workspace_that_is_not_one_piece_is_refused(kernels):
    """The elements between those of a view, and memory behind it, are not the call's."""
    sizes = kernels.kv4_decode_workspace_bytes(8, 2, 128), kernels.gemm_adapters_workspace_bytes(4, 64, 16)
    for call, size in zip((decode, project), sizes):
        room = torch.zeros(2 * size, dtype=torch.uint8, device=DEV)
        with pytest.raises(ValueError, match="contiguous"):
            call(kernels, workspace=room[::2])
        torch.cuda.synchronize()
        assert (room == 0).all()
        assert call(kernels, workspace=room[:size]).isfinite().all()
