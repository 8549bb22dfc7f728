"""The calls of pages_shapes.py reach the forms that they are for (tessera_amd/csrc/launch_rules.hpp: pages_rule)."""
import pages_shapes as shapes
from test_launch_rules import run_program


def test_forms(tmp_path):
    lines, count = [], 0
    for how, pairs, d in shapes.forms():
        group, rows, past, most_rows, most_len = shapes.sizes(how, pairs)
        wanted = {"short": "s.parts == 1 && s.even == 0", "many": "s.parts == 1 && s.even == 0 && s.waves == 4", "parts": "s.parts > 1",
                  "even": "s.even != 0"}[how]
        cols = shapes.columns(pairs, d)
        if how != "parts" and cols is None:
            wanted = "true"                    # (many columns: parts where the units do not fill the chip)
        wanted += f" && s.columns == {cols}" if cols is not None else " && s.columns >= 64"
        if how == "short" and cols is not None:
            wanted += " && s.waves == 8"
        lines.append(f"""{{ const PagesShape s = pages_rule(PagesCall{{{sum(rows)}, {len(rows)}, {group}, {shapes.KV}, {d}, {most_rows}, {most_len}, 0, 0}}, 256, size_t{{16}} << 20);
    CHECK({wanted}, "{how} {pairs} {d}: %zu columns, %zu parts, even %zu, waves %zu", static_cast<size_t>(s.columns), static_cast<size_t>(s.parts),
          static_cast<size_t>(s.even), static_cast<size_t>(s.waves)); }}""")
        count += 1
    assert count > 100
    run_program(tmp_path, "\n  ".join(lines))
