// operators.h — the operator programs: hand-written kernels in the form that
// Emit gives a DSL program (source, launch plan, hipcc arguments).
#ifndef TCA_CG_OPERATORS_H_
#define TCA_CG_OPERATORS_H_

#include <string>

#include "emit.h"

namespace tca {
namespace cg {

enum class OpStatus { Ok, NoSuchOperator, Unsupported };

// `attributes` as include/tca_op.h lists them. On Ok, *program is the name
// the symbols carry (the operator and its attributes).
OpStatus EmitOperator(const std::string& name, const std::string& attributes, const std::string& target, Result* out,
                      std::string* program, std::string* err);

// One line per operator: its name and the attributes it takes.
std::string ListOperators();

}  // namespace cg
}  // namespace tca

#endif  // TCA_CG_OPERATORS_H_
