"""GPU: the camera's refresh and the camera math as recorded launches, replayed against the same calls issued directly."""

import ctypes

import pytest
import torch

from conftest import load_golden
from isaaclab_amd import _abi
from isaaclab_amd.utils.command_list import CommandList

pytestmark = pytest.mark.gpu


def test_a_recorded_camera_refresh(dev):
    from isaaclab_amd.sensors.patterns import PinholeCameraPatternCfg
    from isaaclab_amd.sensors.ray_caster_camera import CameraOffsetCfg, RayCasterCamera, RayCasterCameraCfg
    from isaaclab_amd.utils.mesh import convert_to_mesh

    g = load_golden("ray_caster_camera")
    kinds = ["distance_to_image_plane", "distance_to_camera", "normals"]

    pos = g["view_pos"].to(dev)   # (the simulator's buffer: written in place, where the recorded launch reads it)

    def camera():
        cfg = RayCasterCameraCfg(offset=CameraOffsetCfg(pos=(0.1, -0.05, 0.2), rot=(0.5, -0.5, 0.5, -0.5), convention="ros"), data_types=kinds,
                                 depth_clipping_behavior="max", max_distance=2.5,
                                 pattern_cfg=PinholeCameraPatternCfg(focal_length=24.0, horizontal_aperture=20.955, width=16, height=12))
        cam = RayCasterCamera(cfg, g["view_pos"].shape[0], convert_to_mesh(g["verts"].numpy(), g["tris"].numpy(), str(dev)), dev)
        cam.set_view_pose(pos, g["view_quat"].to(dev))
        return cam

    direct, replayed = camera(), camera()
    assert torch.equal(direct.data.pos_w, replayed.data.pos_w)   # both refreshed once
    commands = CommandList()
    with commands.record():
        replayed._update_outdated_buffers()
    assert len(commands) == 2
    for shift in (0.0, 0.25, -0.1):
        pos.copy_(g["view_pos"].to(dev) + shift)
        direct._is_outdated[:] = replayed._is_outdated[:] = True
        direct._update_outdated_buffers()
        commands.replay()
        torch.cuda.synchronize()
        assert torch.equal(direct._data.pos_w, replayed._data.pos_w) and torch.equal(direct.frame, replayed.frame)
        for kind in kinds:
            a, b = direct._data.output[kind], replayed._data.output[kind]
            assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)), (kind, shift)
        assert not replayed._is_outdated.any()


def test_a_recorded_camera_op(dev):
    depth, K = torch.rand(3, 5, 7, device=dev) + 1, torch.tensor([[[4.0, 0, 3], [0, 5, 2], [0, 0, 1]]], device=dev)
    p, i = ctypes.c_void_p, ctypes.c_int64
    op = lambda out: _abi.check(_abi.lib.ilx_camera_op(0, p(depth.data_ptr()), p(K.data_ptr()), i(1), p(out.data_ptr()), i(3), 5, 7, p(_abi.stream())))  # noqa: E731
    want, got = torch.zeros_like(depth), torch.zeros_like(depth)
    op(want)
    commands = CommandList()
    with commands.record():
        op(got)
    commands.replay()
    assert torch.equal(got, want) and want.abs().sum() > 0
