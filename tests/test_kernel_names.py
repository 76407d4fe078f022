"""Every kernel of the built library is registered under its own name (CPU: nothing is launched).

A kernel whose mangled name differs between the host and the device pass (an argument type that depends on an enumeration
without a name) links, and its first launch ends the process.
"""

from __future__ import annotations

import re
import struct

from test_kernel_resources import kernels, kernels_of  # noqa: F401  (the fixture builds the library where it is missing)

from conftest import load_pkg


def test_every_kernel_is_registered(kernels):  # noqa: F811
    lib = open(load_pkg().library_path(), "rb").read()
    host = bytearray(lib)
    for m in re.finditer(rb"__CLANG_OFFLOAD_BUNDLE__", lib):
        at = m.start()
        pos = at + 32
        for _ in range(struct.unpack_from("<Q", lib, at + 24)[0]):
            off, size, n = struct.unpack_from("<QQQ", lib, pos)
            pos += 24 + n
            host[at + off:at + off + size] = bytes(size)
    names = set(bytes(host).split(b"\0"))
    missing = [k for k in kernels if k.encode() not in names]
    assert not missing, missing[:3]
