"""Calls of the heads that their documentation allows and their ordinary use does not make,
as far as they need no device."""

from __future__ import annotations

from test_host_rules import run_cpp


def test_a_sampling_call_keeps_to_its_workspace(tmp_path):
    """Launches of a call cover its rows, and take tiles only where the call's workspace
    (whose size is asked for with the whole call's rows) holds them: not the last 1 to 128
    rows of a call that takes several launches."""
    run_cpp(tmp_path, """
    const uint64_t launch = 1ull << 21;
    for (uint64_t n : std::vector<uint64_t>{1ull, 5ull, 128ull, 129ull, 4096ull, launch - 1, launch, launch + 1,
                       launch + 128, launch + 129, 3 * launch, 3 * launch + 77, 1ull << 40})
        for (uint32_t v : {1u, 1024u, 16384u, 16385u, 262144u}) {
            const uint64_t held = sample_tiled_rows(n, v);
            CHECK(held == (n <= 128 && v > 16384 ? n : 0));
            uint64_t next = 0;
            sample_launches(n, v, [&](uint64_t r, uint64_t rows, bool tiled) {
                CHECK(r == next && rows >= 1 && rows <= launch);
                CHECK(!tiled || r + rows <= held);
                CHECK(tiled == (held > 0));
                next = r + rows;
            });
            CHECK(next == n);
        }""")
