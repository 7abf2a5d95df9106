# Sourced by the scripts here that compile the library: its sources (without suffix) and its compiler flags, as __graft_entry__.py has them.
ROOT="$(cd "$(dirname "${BASH_SOURCE[0]}")/.." && pwd)"
HIPCC="${HIPCC:-hipcc}"
SRCS="$(cd "$ROOT" && python3 -c 'import __graft_entry__ as g; print(*[s.rsplit(".", 1)[0] for s in g.HIP_SOURCES])')"
FLAGS="$(cd "$ROOT" && python3 -c 'import __graft_entry__ as g; print(*g.HIP_FLAGS)')"
