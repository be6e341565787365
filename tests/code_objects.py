"""The gfx950 code objects inside the built library: what the compiler says of each kernel
(registers, scratch) and its instructions, for tests of properties that no result shows."""
import os
import re
import struct
import subprocess
import tempfile

_MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"
_LLVM = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin")


def _bundled(data):
    """The device images of every bundle in the library's bytes (one a source file)."""
    at = data.find(_MAGIC)
    while at >= 0:
        count, = struct.unpack_from("<Q", data, at + len(_MAGIC))
        entry = at + len(_MAGIC) + 8
        for _ in range(count):
            offset, size, name = struct.unpack_from("<QQQ", data, entry)
            target = data[entry + 24:entry + 24 + name].decode()
            entry += 24 + name
            if target.startswith("hip") and target.endswith("gfx950") and size:
                yield data[at + offset:at + offset + size]
        at = data.find(_MAGIC, entry)


def _tool(name, *args):
    return subprocess.run([os.path.join(_LLVM, name), *args], check=True, capture_output=True,
                          text=True).stdout


def kernels(library, pattern):
    """{kernel: (its metadata's whole numbers, its instructions)} of those whose name holds
    `pattern`."""
    with open(library, "rb") as f:
        images = [x for x in _bundled(f.read()) if pattern.encode() in x]
    out = {}
    for image in images:
        with tempfile.TemporaryDirectory() as d:
            path = os.path.join(d, "code")
            with open(path, "wb") as f:
                f.write(image)
            notes, text = _tool("llvm-readelf", "--notes", path), \
                _tool("llvm-objdump", "-d", "--no-show-raw-insn", path)
        body = {m[0]: m[1].splitlines() for m in
                re.findall(r"^[0-9a-f]+ <(\S+)>:\n(.*?)(?=^\S|\Z)", text, re.M | re.S)}
        for block in re.split(r"^  - ", notes, flags=re.M)[1:]:
            name = re.search(r"\.name:\s+(\S+)", re.sub(r"(?m)^      .*$", "", block))
            if name and pattern in name[1]:
                values = {k: int(v) for k, v in re.findall(r"^ *\.(\w+):\s+(\d+)$", block, re.M)}
                out[name[1]] = values, [x.split("//")[0].strip() for x in body[name[1]] if x.strip()]
    return out
