"""What a command list keeps of a recorded launch: all of the kernel's arguments (no GPU needed).

``ilx::launch`` is a template over the kernels' argument types.  Two types of one name in two files would be one type to the linker, which
keeps a single copy of every function instantiated by it; the launch of the one would then copy the size of the other."""

import ctypes
import os
import re

from isaaclab_amd import _abi
from isaaclab_amd.utils.command_list import CommandList

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "isaaclab_amd", "csrc")


class Vector(ctypes.Structure):
    _fields_ = [("begin", ctypes.c_void_p), ("end", ctypes.c_void_p), ("capacity", ctypes.c_void_p)]


class Command(ctypes.Structure):
    """Mirror of ``ilx::Command`` (csrc/common.h)."""

    _fields_ = [("kernel", ctypes.c_void_p), ("grid", ctypes.c_uint32 * 3), ("block", ctypes.c_uint32 * 3), ("shmem", ctypes.c_uint32),
                ("blob", Vector), ("args", Vector)]


def kept(commands):
    """The bytes of every kept launch's arguments (the library ends them with one byte more)."""
    held = Vector.from_address(commands._handle.value)
    assert held.end - held.begin == len(commands) * ctypes.sizeof(Command)
    found = (Command * len(commands)).from_address(held.begin)
    return [ctypes.string_at(c.blob.begin, c.blob.end - c.blob.begin - 1) for c in found]


def test_a_recorded_camera_keeps_its_arguments():
    commands = CommandList()
    mesh = ctypes.create_string_buffer(b"\x5a" * (1 << 16))
    names = [n for n, kind in _abi.RayCasterCameraDesc._fields_ if kind is ctypes.c_void_p and n not in ("mesh", "timestamp", "timestamp_last_update",
                                                                                                         "is_outdated")]
    pointers = {n: 0x10000 * (k + 1) for k, n in enumerate(names)}
    camera = _abi.RayCasterCameraDesc(mesh=ctypes.addressof(mesh), num_envs=77, num_rays=91, depth_clipping=1, max_distance=2.5, view_pos_stride=13,
                                      view_quat_stride=17, **pointers)
    data, intrinsics, out = 0x7100000, 0x7200000, 0x7300000
    with commands.record():   # (what a call answers without a device does not matter: its launch is kept before)
        _abi.lib.ilx_raycaster_camera_refresh(ctypes.byref(camera), None)
        _abi.lib.ilx_camera_op(0, *map(ctypes.c_void_p, (data, intrinsics)), ctypes.c_int64(1), ctypes.c_void_p(out), ctypes.c_int64(5), 6, 7, None)
    refresh, op = kept(commands)
    for value in pointers.values():
        assert value.to_bytes(8, "little") in refresh, hex(value)
    assert (77).to_bytes(8, "little") + (91).to_bytes(4, "little") in refresh and len(refresh) > 8 * len(pointers) + 16
    for value in (data, intrinsics, out):
        assert value.to_bytes(8, "little") in op
    assert op.endswith((6).to_bytes(4, "little") + (7).to_bytes(4, "little")) and len(op) == 56


def types_of(path):
    """Names of the types defined at namespace scope, but for those in an unnamed namespace."""
    with open(path) as f:
        text = re.sub(r'//[^\n]*|/\*.*?\*/|"(?:\\.|[^"\\])*"|^\s*#[^\n]*(?:\\\n[^\n]*)*', " ", f.read(), flags=re.S | re.M)
    scopes, names, head = [], [], ""
    for token in re.findall(r"[{};]|[^{};]+", text):
        if token == "{":
            space = re.search(r"\bnamespace\s*(\w*)\s*$", head) or (re.search(r'extern\s*$', head) and re.match("()", ""))
            if space:
                scopes.append("unnamed" if head.strip().endswith("namespace") else "named")
            else:
                found = re.search(r"\b(?:struct|class|union|enum)\s+(?:__attribute__\s*\(\(.*?\)\)\)?\s*|alignas\s*\(.*?\)\s*)?(\w+)\s*(?:final\s*)?(?::[^{]*)?$", head)
                if found and all(s == "named" for s in scopes):
                    names.append(found.group(1))
                scopes.append("body")
            head = ""
        elif token == "}":
            scopes.pop()
            head = ""
        elif token == ";":
            head = ""
        else:
            head = token
    assert not scopes, path
    return names


def test_every_type_has_one_name():
    files = sorted(f for f in os.listdir(CSRC) if f.endswith((".hip", ".cpp", ".h")))
    where = {}
    for f in files:
        for name in types_of(os.path.join(CSRC, f)):
            where.setdefault(name, []).append(f)
    assert {"StateSpaceArgs", "ConvArgs", "NormArgs", "Command", "CommandList"} <= set(where)   # (the reading finds what is there)
    assert not {name: found for name, found in where.items() if len(found) > 1}
