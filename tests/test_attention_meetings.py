"""The tree in which blocks put the parts of a group of rows together: every meeting counts its blocks in a word that no other one uses.  The rule is compiled for the host: no
GPU is needed."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tannic_amd", "csrc")

# every meeting of 2 .. 1024 parts, as the kernels go through them (1024: as many as there are words)
PROGRAM = r'''
#include <cstdio>
#include <cstdlib>
#include <map>
#include <utility>
#include "meeting.hpp"
int main(int, char** argument) {
    const uint32_t most = std::atoi(argument[1]);
    for (uint32_t all = 2; all <= 1024; ++all) {
        std::map<uint32_t, std::pair<uint32_t, uint32_t>> used;
        uint32_t level = 0, apart = 1;
        for (uint32_t parts = all; parts > 1; parts = (parts + most - 1) / most, apart *= most, ++level)
            for (uint32_t first = 0; first < parts; first += most) {
                if (parts - first < 2) continue;      // (alone: nothing is counted)
                const uint32_t count = th::meeting_count(first, apart);
                if (count == 0 || count >= all) return std::printf("%u parts, level %u, first %u: word %u\n", all, level, first, count), 1;
                const auto [at, fresh] = used.insert({count, {level, first}});
                if (!fresh) return std::printf("%u parts: level %u, first %u and level %u, first %u share word %u\n", all, level, first, at->second.first, at->second.second, count), 1;
            }
    }
    return 0;
}
'''


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    where = tmp_path_factory.mktemp("meetings")
    source, binary = where / "meetings.cpp", where / "meetings"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC, str(source), "-o", str(binary)], check=True)
    return str(binary)


@pytest.mark.parametrize("most", [2, 4, 8, 16, 32, 64])
def test_no_two_meetings_share_a_word(most, program):
    done = subprocess.run([program, str(most)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout
