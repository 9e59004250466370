// Annotations of gernels that divide one result among the workgroups of a launch
// and read everything else whole: the operators of a serving step.  Nothing in
// the reference corresponds to these.
#pragma once

#include "annot/table.h"

#include <cstdint>
#include <string>
#include <utility>
#include <vector>

namespace gern {
namespace annot {

// A data structure that a function reads whole: no fields, and a query that
// names it.
class WholeADT : public TableADT {
public:
    WholeADT(const std::string &name, const std::string &type)
        : TableADT(name, type) {
        query_call = call("whole");
        free_call = FunctionSignature{};
    }
};

// A data structure that the workgroups of a launch divide among them along one
// or more axes of members that count the pieces.  Fields: the piece's index on
// each axis, then the (constant) number of pieces on each.  Its query names the
// piece; the function writes through it.
template<class Host>
class PiecesADT : public TableADT {
public:
    using Axis = std::pair<std::string, int64_t Host::*>;
    PiecesADT(const std::string &name, const std::string &type, const std::string &query, const std::vector<Axis> &axes)
        : TableADT(name, type), axes(axes) {
        std::vector<Variable> at, extent;
        for (const auto &axis : axes) {
            at.push_back(Variable("at_" + axis.first));
            extent.push_back(Variable("n_" + axis.first, Datatype::Int64, true));
        }
        fields = at;
        fields.insert(fields.end(), extent.begin(), extent.end());
        query_call = call(query, at);
        insert_call = call("unsupported_insert");
        allocate_call = call("unsupported_allocate");
        temporaries_are_freed = false;
    }
    bool readMember(const void *object, const std::string &member, int64_t &value) const override {
        for (const auto &axis : axes) {
            if (axis.first == member) {
                value = static_cast<const Host *>(object)->*axis.second;
                return true;
            }
        }
        return false;
    }

private:
    std::vector<Axis> axes;
};

// A gernel that reads data structures whole and writes a piece of another:
// name<bound...>(whole..., piece).  `bound` are variables that the caller binds.
class PieceFunction : public AbstractFunction {
public:
    PieceFunction(const std::string &name, const std::string &header, const std::vector<AbstractDataTypePtr> &whole,
                  AbstractDataTypePtr out, const std::vector<std::string> &axes, const std::vector<std::string> &bound)
        : name(name), header(header), whole(whole), out(out), axes(axes) {
        for (const auto &b : bound) {
            constants.push_back(Variable(b, Datatype::Int64, true));
        }
    }
    Annotation getAnnotation() override {
        std::vector<Variable> at, extent;
        std::vector<Variable> piece;
        for (const auto &axis : axes) {
            at.push_back(Variable("at_" + axis));
            extent.push_back(Variable("n_" + axis, Datatype::Int64, true));
        }
        piece.insert(piece.end(), at.begin(), at.end());
        piece.insert(piece.end(), extent.begin(), extent.end());
        std::vector<SubsetObj> reads;
        for (const auto &ds : whole) {
            reads.push_back(SubsetObj(ds, {}));
        }
        Pattern annotation = Tileable(at.back() = Expr(0), ADTMember(out, axes.back(), false), extent.back(),
                                      Produces::Subset(out, piece), Consumes::Subsets(SubsetObjMany(reads)));
        for (size_t i = axes.size() - 1; i-- > 0;) {
            annotation = Tileable(at[i] = Expr(0), ADTMember(out, axes[i], false), extent[i], annotation);
        }
        return annotation.occupies({Grid::Unit::THREAD_X});
    }
    FunctionSignature getFunction() override {
        FunctionSignature f;
        f.name = name;
        for (const auto &ds : whole) {
            f.args.push_back(Parameter(ds));
        }
        f.args.push_back(Parameter(out));
        f.template_args = constants;
        return f;
    }
    std::vector<std::string> getHeader() override {
        return {header};
    }

private:
    std::string name, header;
    std::vector<AbstractDataTypePtr> whole;
    AbstractDataTypePtr out;
    std::vector<std::string> axes;
    std::vector<Variable> constants;
};

}  // namespace annot
}  // namespace gern
