"""From how many slots on a routing call writes its workspace: what the header promises is what the launches do (text and host arithmetic, no GPU)."""
import os
import re

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))


def source(*path):
    with open(os.path.join(ROOT, *path)) as f:
        return f.read()


def constants():
    text = source("grouped_mm_bf16_amd", "csrc", "gmm_moe.hip")
    value = lambda name: int(re.search(rf"constexpr int {name} = (\d+);", text).group(1))
    waves = value("kPlaceWaves")
    assert re.search(r"constexpr int kPlaceBlock = 64 \* kPlaceWaves;", text)
    return value("kCountedSlots"), value("kPlaceSlots"), 64 * waves * value("kMaxSortBlocks")


def comment_before(text, name):
    at = text.index(f"int {name}(")
    return " ".join(re.sub(r"\n \* ?", " ", text[text.rindex("/*", 0, at):at]).split())


def test_header_and_launches_agree():
    counted, placed, tabled = constants()
    header = source("include", "grouped_mm_hip.h")
    shared, own, none = (comment_before(header, name) for name in ("gmm_moe_route", "gmm_moe_route_own", "gmm_moe_route_noalloc"))
    assert f"two for up to {placed} slots, three for up to {tabled}, four for more" in shared
    assert f"Calls of up to {placed} slots leave the workspace alone" in shared
    assert f"written from {counted + 1} slots on" in own and f"two launches for up to {counted} slots, three for up to {tabled}, four for more" in own
    assert f"more than {placed} slots share that array" in none


def test_which_call_has_a_table_of_its_own():
    text = source("grouped_mm_bf16_amd", "csrc", "gmm_moe.hip")
    for name, shared in (("gmm_moe_route", "true"), ("gmm_moe_route_own", "false"), ("gmm_moe_route_noalloc", "true")):
        body = text[text.index(f"int {name}("):]
        assert re.search(r"route_checked\([^;]*, (true|false),\s*static_cast<hipStream_t>\(stream\)\);", body).group(1) == shared, name
    assert re.search(r"pl\.slots > kCountedSlots && blocks <= pl\.nb && !\(table_shared && pl\.slots <= kPlaceSlots\)", text)
