"""The C++ nodes of the attention and the cache hand every operand to its place: compiled over a stand-in of the front end, with the library's entry points replaced."""
import subprocess

import adapter_build


def test_the_nodes_hand_over_what_they_were_given(tmp_path):
    binary = adapter_build.build(str(tmp_path), "-DRECORD")
    (tmp_path / "none").write_bytes(b"")
    done = subprocess.run([binary, str(tmp_path / "none"), str(tmp_path / "out")], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stderr
    # q k v lengths: 1 .. 4, their results 5 and 6; keys values k v q cos sin: 7 .. 13, table starts context: 14 .. 16, the turned queries 17, the attention 18
    assert done.stdout.splitlines() == [
        "attend 1 2 3 0 5 stream 77 scale 0.25",
        "attend 1 2 3 4 6 stream 77 scale -0.5",
        "append_pages 9 10 14 15 16 0 0 0 7 8 0 stream 77",
        "append_pages 9 10 14 15 16 12 13 11 7 8 17 stream 77",
        "attend_pages 11 7 8 14 15 16 18 stream 77 scale 0.125",
        "copy_pages 7 stream 77 1>5 5>2",
        "host: attend: implemented by the device backend only (move the operands to a Device)",
        "mixed: attend_pages: operands live in different environments",
        "lists: copy_pages: as many sources as targets",
        "attend 1 2 3 0 19 stream 77 scale 1",
        "types: attend: unsupported dtype",
        "append_pages 9 10 14 15 16 0 0 0 7 8 0 stream 77",
        "refused: append_pages: rejected by the device backend (shapes or dtypes do not fit)",
    ]
