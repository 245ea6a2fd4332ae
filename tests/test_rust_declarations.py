"""CPU checks of the documented Rust declarations against the C header: every
type that they use is declared, the structs have the header's fields in its
order, and the constants its values."""
from __future__ import annotations

import ctypes as C
import re
from pathlib import Path

from bobcat_amd._lib import KvShape, LogitRules
from bobcat_amd.backend import LOGIT_ROW, NO_MASK

ROOT = Path(__file__).resolve().parent.parent
HEADER = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "bobcat_hip.h").read_text(), flags=re.S)
RUST = re.sub(r"//.*", "", "\n".join(block for path in sorted(ROOT.glob("*.md"))
                                      for block in re.findall(r"```rust\n(.*?)```", path.read_text(), re.S)))


def c_structs():
    """Field names (and their types) of the header's structs by their Rust names."""
    out = {}
    for name, body in re.findall(r"typedef struct (\w+) \{(.*?)\}", HEADER, re.S):
        fields = []
        for line in body.split(";"):
            parts = line.replace("\n", " ").strip()
            if parts:
                kind, names = re.match(r"((?:const )?\w+ ?\**)(.*)", parts).groups()
                fields += [(kind.strip(), n.strip(" *")) for n in names.split(",")]
        out["".join(p.capitalize() for p in name.split("_"))] = fields
    return out


def rust_structs():
    return {name: [(f.split(":")[1].strip(), f.split(":")[0].strip()) for f in re.findall(r"pub (\w+: [^,\n}]+)", body)]
            for name, body in re.findall(r"pub struct (Bch\w+) \{(.*?)\}", RUST, re.S)}


def test_every_type_is_declared():
    used = set(re.findall(r"\bBch[A-Z]\w*", RUST))
    assert used and used <= set(rust_structs()), used - set(rust_structs())


def test_structs_have_the_headers_fields():
    kinds = {"uint32_t": "u32", "uint64_t": "u64", "float": "f32", "bch_view": "BchView"}
    rust = rust_structs()
    for name in ("BchKvShape", "BchLogitRow", "BchLogitRules", "BchSampling"):
        assert rust[name] == [(kinds[kind], field) for kind, field in c_structs()[name]], name


def test_sizes_of_the_serving_structs():
    assert C.sizeof(KvShape) == 20 and C.sizeof(LogitRules) == 96 and LOGIT_ROW.itemsize == 32
    assert [f for _, f in c_structs()["BchKvShape"]] == [f for f, _ in KvShape._fields_]
    assert [f for _, f in c_structs()["BchLogitRules"]] == [f for f, _ in LogitRules._fields_]
    assert [f for _, f in c_structs()["BchLogitRow"]] == list(LOGIT_ROW.names)


def test_constants():
    rust = dict(re.findall(r"pub const (BCH_\w+): u32 = (\w+);", RUST))
    assert int(rust["BCH_NO_MASK"], 16) == NO_MASK
    for name in ("BCH_KV_F16", "BCH_KV_I8", "BCH_KV_F8"):
        assert rust[name] == re.search(rf"{name} = (\d+)", HEADER)[1]
