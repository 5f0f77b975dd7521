"""Checks the machine code of the many-row dense products (csrc/mxfp4_gemm.cuh) for what their inline assembly takes on itself.

The compiler knows neither that the products written there deliver their sums late nor that the requests beside them count towards the
waits, so nothing of its own keeps these rules; the build does, by reading what it made:

  sums        nothing but a product touches an accumulator register within 12 wait states behind the product that writes it
  operands    a vector register that a product reads has not been written by a vector instruction in the two wait states before it
  requests    a copy into LDS reads no scalar register that a vector instruction wrote in the five wait states before it, and
              m0 is written at least one before it, by scalar moves alone
  counting    there is no other load from memory, and none through scratch memory: the waits count the requests, in order
  stores      tiles stored while the next one's requests are in flight are stored by as many instructions as the waits count
"""
import os
import re
import struct
import subprocess
import tempfile

OBJDUMP = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-objdump")
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"
KERNEL = "tf_mx_gemm"
SUM_STATES, OPERAND_STATES, SCALAR_STATES, M0_STATES = 12, 2, 5, 1
PERSISTENT_STORES = 32          # FM * FT / 2 of the 256 x 256 tiles


def device_images(path):
    """The gfx950 code objects inside a host object or library: bundles of (count, then offset, size and name of each entry)."""
    data, images, at = open(path, "rb").read(), [], 0
    while (at := data.find(MAGIC, at)) >= 0:
        count, place = struct.unpack_from("<Q", data, at + 24)[0], at + 32
        for _ in range(count):
            offset, size, length = struct.unpack_from("<QQQ", data, place)
            name = data[place + 24:place + 24 + length].decode()
            place += 24 + length
            if name.endswith("gfx950") and size:
                images.append(data[at + offset:at + offset + size])
        at += len(MAGIC)
    return images


def disassemble(image):
    with tempfile.TemporaryDirectory() as folder:
        file = os.path.join(folder, "image.co")
        with open(file, "wb") as f:
            f.write(image)
        return subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", file], check=True, stdout=subprocess.PIPE, text=True).stdout


class Instruction:
    __slots__ = ("address", "name", "text", "operands", "target", "states")

    def __init__(self, address, text, target):
        self.address, self.text, self.target = address, text, target
        self.name, _, rest = text.partition(" ")
        self.operands = [_registers(o) for o in re.split(r",\s*(?![^\[]*\])", rest)] if rest else []
        self.states = int(rest, 0) + 1 if self.name == "s_nop" else 1

    @property
    def product(self):
        return self.name.startswith("v_mfma")

    @property
    def vector(self):
        return self.name.startswith("v_") and not self.product

    @property
    def request(self):
        return self.name.startswith("global_load_lds")

    def written(self):
        """Registers that a vector instruction writes (two of them where it swaps or carries)."""
        both = 2 if "swap" in self.name or "_co_" in self.name or "div_scale" in self.name else 1
        written = set().union(*self.operands[:both]) if self.operands else set()
        return written | ({"vcc"} if self.name.startswith("v_cmp") and "e32" in self.name else set())


def _registers(operand):
    """{"v3", "a7", "s12", "vcc", "m0"} of an operand's text."""
    out = set(re.findall(r"\b(?:vcc|m0|exec)\b", operand))
    for kind, first, last in re.findall(r"\b([vas])\[(\d+):(\d+)\]", operand):
        out |= {kind + str(i) for i in range(int(first), int(last) + 1)}
    return out | set(re.findall(r"(?<![\w\[:])([vas]\d+)\b", operand))


def kernels(listing, name=KERNEL):
    """{symbol: [Instruction]} of the listing's functions whose symbol contains `name`."""
    found, now, base = {}, None, 0
    for line in listing.splitlines():
        head = re.match(r"([0-9a-f]+) <(\S+)>:", line)
        if head:
            base, symbol = int(head.group(1), 16), head.group(2)
            now = found.setdefault(symbol, []) if name in symbol else None
        elif now is not None and line.startswith("\t"):
            text, _, comment = line.partition("//")
            address = re.match(r"\s*([0-9A-F]+):", comment)
            if not address:
                continue                                             # "...": zeros behind the code
            target = re.search(r"<[^>+]+(?:\+0x([0-9a-f]+))?>", comment) if re.match(r"\s*s_c?branch", text) else None
            now.append(Instruction(int(address.group(1), 16), " ".join(text.split()), base + int(target.group(1) or "0", 16) if target else None))
    return found


def _before(code, preceding, at, states):
    """Every instruction that some path runs fewer than `states` wait states before instruction `at`."""
    seen, todo = {}, [(j, 0) for j in preceding[at]]
    while todo:
        j, passed = todo.pop()
        if passed >= states or seen.get(j, states) <= passed:
            continue
        seen[j] = passed
        todo += [(i, passed + code[j].states) for i in preceding[j]]
    return [code[j] for j in seen]


def faults(code):
    """What the instructions of one kernel break, as texts."""
    place = {c.address: i for i, c in enumerate(code)}
    preceding = [[i - 1] if i and code[i - 1].name not in ("s_branch", "s_endpgm", "s_setpc_b64") else [] for i in range(len(code))]
    for i, c in enumerate(code):
        if c.target is not None:
            preceding[place[c.target]].append(i)
    out = []

    def fault(rule, c, other):
        out.append("%s: %s at %x behind %s at %x" % (rule, c.text, c.address, other.text, other.address))

    for i, c in enumerate(code):
        used = set().union(*c.operands) if c.operands else set()
        if c.product:
            read = set().union(*c.operands[1:])
            for b in _before(code, preceding, i, OPERAND_STATES):
                if b.vector and b.written() & read:
                    fault("operands", c, b)
        elif any(r[0] == "a" and r[1:].isdigit() for r in used):
            for b in _before(code, preceding, i, SUM_STATES):
                if b.product and b.operands[0] & used:
                    fault("sums", c, b)
        if c.request:
            for b in _before(code, preceding, i, SCALAR_STATES):
                if b.vector and any(r[0] == "s" for r in b.written() & used):
                    fault("requests", c, b)
            for b in _before(code, preceding, i, M0_STATES):
                if b.operands and "m0" in b.operands[0]:
                    fault("requests", c, b)
        elif "m0" in used and c.name != "s_mov_b32":
            out.append("requests: m0 in %s at %x" % (c.text, c.address))
        elif c.name.startswith("scratch_") or re.match(r"(global|flat|buffer)_(load|atomic)", c.name):
            out.append("counting: %s at %x" % (c.text, c.address))
    stores = [c for c in code if c.name.startswith("buffer_store")]
    if stores and (len(stores) != PERSISTENT_STORES or any(re.match(r"(global|flat)_store", c.name) for c in code)):
        out.append("stores: %d instead of %d" % (len(stores), PERSISTENT_STORES))
    return out


def check(path):
    """The number of many-row product kernels in a host object or library; RuntimeError where one breaks a rule."""
    found = {}
    for image in device_images(path):
        found.update(kernels(disassemble(image)))
    broken = {name: f for name, code in found.items() if (f := faults(code))}
    if broken:
        raise RuntimeError("%s:\n%s" % (path, "\n".join("%s: %d\n  %s" % (name, len(f), "\n  ".join(f[:4])) for name, f in broken.items())))
    return len(found)
