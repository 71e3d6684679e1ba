"""CPU: what the entries of cross attention, RMS norm and gradient clipping, and the trainer around them, decide on the host."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_nothing_turns_graph_packet_capture_on():
    """with it replayed graphs end in a GPU memory fault: no tool, benchmark or module sets the variable to anything but 0"""
    for folder in ("", "tools", "ogmm_amd", "perf", "oracle"):
        for name in sorted(os.listdir(os.path.join(ROOT, folder))):
            if name.endswith((".py", ".sh")):
                text = open(os.path.join(ROOT, folder, name), encoding="utf-8").read()
                assert not re.search(r"PACKET_CAPTURE\W{0,8}=\W{0,3}[1-9]", text), os.path.join(folder, name)
