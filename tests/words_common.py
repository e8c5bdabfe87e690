"""Imported before scan2cap_amd.word_ops: builds the library and the operators' binding where neither is there."""
import os

from scan2cap_amd import build

if not os.path.exists(build.EXT_PATH):
    build.build()
    build.build_ext()
