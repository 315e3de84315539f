"""Workspaces of the serving operators: what the bindings accept (no GPU)."""
import pytest
import torch

from trinity_lowering import kernels as k


@pytest.mark.parametrize("view", [lambda t: t[::2], lambda t: t[:1].expand(1 << 20), lambda t: t.view(64, 64)[:, :32], lambda t: t.view(64, 64).t()])
def test_a_workspace_that_is_not_one_piece_is_refused(view):
    """Its bytes would lie between and behind those of the view."""
    room = torch.empty(4096, dtype=torch.uint8)
    with pytest.raises(ValueError, match="contiguous"):
        k._workspace_operand(view(room), room.get_device(), "kv4_decode")
    k._workspace_operand(room[16:64], room.get_device(), "kv4_decode")
    with pytest.raises(ValueError, match="device"):
        k._workspace_operand(room, 0, "kv4_decode")
