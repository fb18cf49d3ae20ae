"""Table entries below 0, which a pool leaves where it had no page: no kernel may form an address
from one (CPU: the source is checked, since what such an address reads or writes lies outside the
arena)."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "stride_amd", "csrc")


def source(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


def test_rows_without_a_page_are_not_written():
    text = source("tc_epilogue.hpp")
    assert len(re.findall(r"\btable\[", text)) == 1 and len(re.findall(r"kv_row\(o,", text)) == 1
    assert re.search(r"if \(kind != 0\) block = o\.kv\.table\[", text)
    assert re.search(r"else if \(block >= 0\) \{\s*uint16_t\* dst = kv_row\(o,", text)
    assert re.search(r"block = kv\.table\[[^;]*;\s*if \(block < 0\) return;", source("exact.hip"))


def test_attention_reads_inside_the_arena():
    """Every table entry that tc_aux.hip reads is raised to 0 where it is read or where it is used."""
    text = source("tc_aux.hip")
    reads = re.findall(r"(max\()?\b(?:p\.kv\.)?table\[[^;]*;", text)
    assert len(reads) == 3
    assert "int block = max(p.kv.table[" in text and "btab[i] = max(p.kv.table[" in text
    assert re.search(r"block = max\(kOwn \? blk\[", text)
